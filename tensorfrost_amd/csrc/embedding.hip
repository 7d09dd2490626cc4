// Embedding lookup with scaling, and the gradient of its table.
//
//   out[i, :] = scale * table[tokens[i], :]            (zeros where tokens[i] lies outside [0, vocab))
//   dtable[v, :] = scale * sum over i with tokens[i] == v of dy[i, :], every row of dtable written
//
// In the reference this is a load with a computed index (TensorFrost/Compiler/Implementations.cpp:451-488 shows the
// remaps) and, backward, an atomic scatter-add of floats, whose result changes with the order in which the adds land.
// Here the positions are brought into the order of their tokens first (stable), and each row of the gradient is a sum
// in the order of the positions, cut at fixed places: it comes out the same every time. Both directions are bound by
// memory: the lookup reads the distinct rows and writes n rows, the gradient reads n rows and writes the whole table.

#include "common.h"

namespace tfhip {

// ---- rows and lanes ------------------------------------------------------------------------------

// A row is moved by `lanes` neighbouring lanes of a wave (a power of two up to 64), VEC floats each, in as many steps as
// it takes; a wave moves 64 / lanes rows side by side. Wide rows keep whole waves and 16-byte accesses; narrow ones
// would leave most lanes idle in that form.
struct RowShape {
	int vec;
	int lanes;
};
static RowShape row_shape(size_t cols, const void* a, const void* b) {
	const uintptr_t at = (uintptr_t)a | (uintptr_t)b;
	RowShape r;
	r.vec = cols % 4 == 0 && at % 16 == 0 ? 4 : cols % 2 == 0 && at % 8 == 0 ? 2 : 1;
	const size_t steps = (cols + r.vec - 1) / r.vec;
	r.lanes = 1;
	while (r.lanes < 64 && (size_t)r.lanes < steps) r.lanes *= 2;
	return r;
}

template <int VEC>
struct Floats {
	typedef float type __attribute__((ext_vector_type(VEC)));
};
template <>
struct Floats<1> {
	typedef float type;
};

// ---- lookup ----------------------------------------------------------------------------------------

// Bound by memory: 65536 x 1024 over 32768 rows 62 us for 397 MB through HBM, 6.4 TB/s. The rows are written past the caches, which
// keep the table's.
constexpr int kLookupRows = 8;  // rows a lane has in flight

template <int VEC>
__global__ __launch_bounds__(256) void embedding_kernel(const int32_t* __restrict__ tokens, const float* __restrict__ table, float* __restrict__ out, size_t n, size_t vocab, size_t cols,
                                                        float scale, int lanes) {
	typedef typename Floats<VEC>::type Vec;
	const int lane = threadIdx.x & (lanes - 1);
	const size_t per_group = 256 / lanes;  // rows side by side
	for (size_t first = (size_t)blockIdx.x * per_group * kLookupRows + threadIdx.x / lanes; first < n; first += (size_t)gridDim.x * per_group * kLookupRows) {
		const float* src[kLookupRows];
		bool known[kLookupRows];
#pragma unroll
		for (int u = 0; u < kLookupRows; u++) {
			const size_t i = first + u * per_group;
			const int32_t t = i < n ? tokens[i] : -1;
			known[u] = t >= 0 && (size_t)t < vocab;
			src[u] = table + (known[u] ? (size_t)t : 0) * cols;
		}
		for (size_t c = (size_t)lane * VEC; c < cols; c += (size_t)lanes * VEC) {
			Vec v[kLookupRows];
#pragma unroll
			for (int u = 0; u < kLookupRows; u++) v[u] = *reinterpret_cast<const Vec*>(src[u] + c);
#pragma unroll
			for (int u = 0; u < kLookupRows; u++) {
				const size_t i = first + u * per_group;
				if (i < n) __builtin_nontemporal_store(known[u] ? v[u] * scale : Vec(0.0f), reinterpret_cast<Vec*>(out + i * cols + c));
			}
		}
	}
}

// ---- the order of the positions ----------------------------------------------------------------------

// Up to kAllPairs positions by counting: the place of position i is the number of keys that are smaller, or equal and
// earlier. A key is the token read as unsigned: what names no row (negative, or beyond the table) is at least vocab and comes
// last. A group places 64 positions, one per lane of each of its waves; the waves each compare them with their share of
// the keys: a lane broadcast, a compare and an add per pair. 2049 positions 7 us, 4096 9 to 11, 8192 16 (the kernels below: 4096 15,
// 8192 16).
constexpr uint32_t kAllPairs = 4096;
constexpr int kCountWaves = 16;
__global__ __launch_bounds__(kCountWaves * 64) void embedding_count_kernel(const uint32_t* __restrict__ tokens, uint32_t* __restrict__ keys, uint32_t* __restrict__ order, uint32_t n) {
	__shared__ uint32_t counts[kCountWaves][64];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const uint32_t my_block = blockIdx.x, mine = my_block * 64 + lane;
	const uint32_t k = mine < n ? tokens[mine] : 0;
	uint32_t before = 0;
	for (uint32_t b0 = wave; b0 * 64 < n; b0 += 4 * kCountWaves) {
		uint32_t other[4];  // four blocks of 64 keys, one key per lane
#pragma unroll
		for (int u = 0; u < 4; u++) {
			const uint32_t at = (b0 + u * kCountWaves) * 64 + lane;
			other[u] = at < n ? tokens[at] : 0xFFFFFFFFu;  // smaller than nothing, and behind every position
		}
#pragma unroll
		for (int u = 0; u < 4; u++) {
			const uint32_t b = b0 + u * kCountWaves;
			if (b * 64 >= n) break;
			if (b < my_block) {  // equal keys count: they stand before
#pragma unroll
				for (int j = 0; j < 64; j++) before += (uint32_t)__builtin_amdgcn_readlane(other[u], j) <= k;
			} else {
#pragma unroll
				for (int j = 0; j < 64; j++) before += (uint32_t)__builtin_amdgcn_readlane(other[u], j) < k;
				if (b == my_block) {
#pragma unroll
					for (int j = 0; j < 64; j++) before += (uint32_t)__builtin_amdgcn_readlane(other[u], j) == k && j < lane;
				}
			}
		}
	}
	counts[wave][lane] = before;
	__syncthreads();
	if (wave == 0 && mine < n) {
		uint32_t at = 0;
#pragma unroll
		for (int w = 0; w < kCountWaves; w++) at += counts[w][lane];
		keys[at] = k;
		order[at] = mine;
	}
}

// Up to kMostTiled positions by a stable sort on 8-bit digits, as many as the table's size has, in tiles of kDigitTile
// small enough that a few tens of thousands of positions spread over the chip (the library's sort, with its tiles of 16384,
// takes 14 us a pass whatever little it is given, and clears and scans its counters in launches of their own; us for the order of
// 16384, 65536, 131072 and 262144 positions over 50257 rows: 17, 25, 34 and 51, the library's sort 39, 45, 46 and 48). Counts are
// kept per tile and digit; a group finds where its keys of a digit go by adding up all tiles' counts itself. (Counting the
// next digit while this pass's keys are written, by atomics, saves a launch of 4.8 us and costs 13: the frequent tokens meet on
// a few counters.)
constexpr uint32_t kDigitTile = 1024, kMostTiled = 131072;

__device__ __forceinline__ uint32_t known_key(int32_t t, uint32_t vocab) { return t >= 0 && (uint32_t)t < vocab ? (uint32_t)t : vocab; }

// counts[tile][256] of one digit; FIRST reads the tokens.
template <bool FIRST>
__global__ __launch_bounds__(256) void embedding_digits_kernel(const int32_t* __restrict__ tokens, const uint32_t* __restrict__ keys, uint32_t* __restrict__ counts, uint32_t n, uint32_t vocab,
                                                               int shift) {
	__shared__ uint32_t count[256];
	count[threadIdx.x] = 0;
	__syncthreads();
#pragma unroll
	for (int j = 0; j < 4; j++) {
		const uint32_t i = blockIdx.x * kDigitTile + j * 256 + threadIdx.x;
		if (i < n) atomicAdd(&count[((FIRST ? known_key(tokens[i], vocab) : keys[i]) >> shift) & 255u], 1u);
	}
	__syncthreads();
	counts[blockIdx.x * 256 + threadIdx.x] = count[threadIdx.x];
}

// One pass: keys and positions to their places by digit `shift / 8`; FIRST reads the tokens.
template <bool FIRST>
__global__ __launch_bounds__(256) void embedding_scatter_kernel(const int32_t* __restrict__ tokens, const uint32_t* __restrict__ keys_in, const uint32_t* __restrict__ order_in,
                                                                uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order_out, const uint32_t* __restrict__ counts, uint32_t n,
                                                                uint32_t vocab, uint32_t tiles, int shift) {
	__shared__ uint32_t wave_count[4][256];
	__shared__ uint32_t place[256];
	__shared__ uint32_t wave_total[4];
	const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	// wave w owns positions [256 w, 256 w + 256) of the tile; item j of lane l is number 64 j + l of them
	const uint32_t base = blockIdx.x * kDigitTile + wave * 256 + lane;
	uint32_t key[4], from[4];
#pragma unroll
	for (int j = 0; j < 4; j++) {
		const uint32_t i = base + j * 64;
		key[j] = i < n ? (FIRST ? known_key(tokens[i], vocab) : keys_in[i]) : 0xFFFFFFFFu;
		from[j] = FIRST ? i : i < n ? order_in[i] : 0u;
	}
#pragma unroll
	for (int w = 0; w < 4; w++) wave_count[w][tid] = 0;
	// keys of digit `tid` in the tiles before this one, and in all
	uint32_t before = 0, total = 0;
	for (uint32_t t0 = 0; t0 < tiles; t0 += 8) {
		uint32_t c[8];
#pragma unroll
		for (int u = 0; u < 8; u++) c[u] = t0 + u < tiles ? counts[(t0 + u) * 256 + tid] : 0u;
#pragma unroll
		for (int u = 0; u < 8; u++) {
			total += c[u];
			before += t0 + u < blockIdx.x ? c[u] : 0u;
		}
	}
	uint32_t upto = total;
#pragma unroll
	for (int off = 1; off < 64; off <<= 1) {
		const uint32_t o = __shfl_up(upto, off, 64);
		if (lane >= off) upto += o;
	}
	if (lane == 63) wave_total[wave] = upto;
	__syncthreads();
	for (int w = 0; w < wave; w++) upto += wave_total[w];
	place[tid] = upto - total + before;
	// the rank of a key among those of its digit in its wave, in the order of the positions
	uint32_t rank[4];
#pragma unroll
	for (int j = 0; j < 4; j++) {
		const uint32_t d = (key[j] >> shift) & 255u;
		uint64_t peers = __ballot(base + j * 64 < n);
#pragma unroll
		for (int b = 0; b < 8; b++) {
			const bool bit = (d >> b) & 1u;
			const uint64_t votes = __ballot(bit);
			peers &= bit ? votes : ~votes;
		}
		const uint32_t ahead = __popcll(peers & ((1ull << lane) - 1));
		const uint32_t seen = wave_count[wave][d];  // read by all peers before the last of them raises it
		__builtin_amdgcn_wave_barrier();
		if (base + j * 64 < n && ahead + 1 == (uint32_t)__popcll(peers)) wave_count[wave][d] = seen + ahead + 1;
		__builtin_amdgcn_wave_barrier();
		rank[j] = seen + ahead;
	}
	__syncthreads();
#pragma unroll
	for (int j = 0; j < 4; j++) {
		if (base + j * 64 >= n) continue;
		const uint32_t d = (key[j] >> shift) & 255u;
		uint32_t at = place[d] + rank[j];
		for (int w = 0; w < wave; w++) at += wave_count[w][d];
		keys_out[at] = key[j];
		order_out[at] = from[j];
	}
}

// For the library's sort, which takes more positions: keys[i] as above, order[i] = i.
__global__ __launch_bounds__(256) void embedding_keys_kernel(const int32_t* __restrict__ tokens, uint32_t* __restrict__ keys, uint32_t* __restrict__ order, uint32_t n, uint32_t vocab) {
	const uint32_t i = blockIdx.x * 256 + threadIdx.x;
	if (i >= n) return;
	keys[i] = known_key(tokens[i], vocab);
	order[i] = i;
}

// ---- sums ----------------------------------------------------------------------------------------------

// First place in the sorted keys that holds at least `key`.
__device__ __forceinline__ uint32_t first_at_least(const uint32_t* __restrict__ keys, uint32_t n, uint32_t key) {
	uint32_t lo = 0, hi = n;
	while (lo < hi) {
		const uint32_t mid = lo + (hi - lo) / 2;
		if (keys[mid] < key)
			lo = mid + 1;
		else
			hi = mid;
	}
	return lo;
}

// The sorted positions are cut into segments of `segment`; `lanes` lanes add up the rows of one segment for the columns
// they own. A run of equal keys that lies in one segment is finished there; the part of a longer run goes to `partial`:
// [segment][0] what continues from the segment before (or fills the segment), [segment][1] what begins here and goes on.
// Bound by memory: 65536 x 1024 into 32768 rows 77 us for 397 MB, 5.1 TB/s.
// The groups behind those of the segments write zeros into the rows that no position names, kZeroRows rows a wave:
// whether a row is named is found by a search for it, all rows of a wave at once.
constexpr int kSumRows = 8, kZeroRows = 8;

template <int VEC>
__global__ __launch_bounds__(256) void embedding_sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order, const float* __restrict__ dy, float* __restrict__ dtable,
                                                            float* __restrict__ partial, uint32_t n, uint32_t vocab, size_t cols, float scale, uint32_t segment, uint32_t segments,
                                                            int lanes, uint32_t col_steps, uint32_t sum_groups) {
	typedef typename Floats<VEC>::type Vec;
	if (blockIdx.x < sum_groups) {
		// unit: a segment and a stretch of lanes * VEC columns; units of one segment are neighbours
		const uint64_t unit = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / (uint32_t)lanes;
		const uint32_t s = (uint32_t)(unit / col_steps);
		const size_t c = ((size_t)(unit % col_steps) * lanes + (threadIdx.x & (lanes - 1))) * VEC;
		if (s >= segments || c >= cols) return;
		const uint32_t begin = s * segment, end = n - begin < segment ? n : begin + segment;
		uint32_t key = keys[begin];
		if (key >= vocab) return;  // positions without a row come last
		bool open = begin > 0 && keys[begin - 1] == key;  // the run began in an earlier segment
		Vec sum = Vec(0.0f);
		uint32_t k[kSumRows], next_k[kSumRows], next_row[kSumRows];
		auto look_up = [&](uint32_t p0) {
#pragma unroll
			for (int u = 0; u < kSumRows; u++) {
				const uint32_t p = p0 + u < end ? p0 + u : end - 1;
				next_k[u] = keys[p];
				next_row[u] = order[p];
			}
		};
		look_up(begin);
		for (uint32_t p0 = begin; p0 < end; p0 += kSumRows) {
			Vec v[kSumRows];
#pragma unroll
			for (int u = 0; u < kSumRows; u++) {
				k[u] = next_k[u];
				v[u] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(dy + (size_t)next_row[u] * cols + c));
			}
			if (p0 + kSumRows < end) look_up(p0 + kSumRows);  // on its way while these rows arrive
#pragma unroll
			for (int u = 0; u < kSumRows; u++) {
				if (p0 + u >= end) break;
				if (k[u] != key) {
					if (open)
						*reinterpret_cast<Vec*>(partial + (size_t)s * 2 * cols + c) = sum;
					else if (key < vocab)
						__builtin_nontemporal_store(sum * scale, reinterpret_cast<Vec*>(dtable + (size_t)key * cols + c));
					open = false;
					key = k[u];
					sum = Vec(0.0f);
				}
				sum += v[u];
			}
		}
		const bool goes_on = end < n && keys[end] == key;
		if (open)
			*reinterpret_cast<Vec*>(partial + (size_t)s * 2 * cols + c) = sum;
		else if (goes_on)
			*reinterpret_cast<Vec*>(partial + ((size_t)s * 2 + 1) * cols + c) = sum;
		else if (key < vocab)
			__builtin_nontemporal_store(sum * scale, reinterpret_cast<Vec*>(dtable + (size_t)key * cols + c));
		return;
	}
	const int lane = threadIdx.x & 63;
	const uint64_t step = (uint64_t)(gridDim.x - sum_groups) * 4 * kZeroRows;
	for (uint64_t v0 = ((uint64_t)(blockIdx.x - sum_groups) * 4 + (threadIdx.x >> 6)) * kZeroRows; v0 < vocab; v0 += step) {
		bool idle = false;
		if (lane < kZeroRows && v0 + lane < vocab) {
			const uint32_t v = (uint32_t)v0 + lane, at = first_at_least(keys, n, v);
			idle = at >= n || keys[at] != v;
		}
		uint64_t rows = __ballot(idle);
		while (rows) {
			const int r = __builtin_ctzll(rows);
			rows &= rows - 1;
			float* to = dtable + (size_t)(v0 + r) * cols;
			for (size_t c = (size_t)lane * VEC; c < cols; c += 64 * VEC) __builtin_nontemporal_store(Vec(0.0f), reinterpret_cast<Vec*>(to + c));
		}
	}
}

// Runs that go over segments: the group of the segment in which such a run begins adds the parts in the order of the
// segments, each wave every eighth one of them for 64 VEC columns, then the waves' sums in the order of the waves.
constexpr int kJoinWaves = 8;
template <int VEC>
__global__ __launch_bounds__(kJoinWaves * 64) void embedding_join_kernel(const uint32_t* __restrict__ keys, float* __restrict__ dtable, const float* __restrict__ partial, uint32_t n,
                                                                         uint32_t vocab, size_t cols, float scale, uint32_t segment, uint32_t segments) {
	typedef typename Floats<VEC>::type Vec;
	__shared__ Vec sums[kJoinWaves][64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const uint32_t s = blockIdx.x;  // the last segment has no run that goes on
	const uint32_t begin = s * segment, end = begin + segment;
	const uint32_t key = keys[end - 1];
	if (keys[end] != key || key >= vocab) return;
	if (begin > 0 && keys[begin - 1] == key) return;  // began earlier: the run fills this segment
	// segments behind this one that begin inside the run
	uint32_t parts = 0;
	for (;;) {
		const uint64_t next = (uint64_t)s + 1 + parts + lane;
		const uint64_t inside = __ballot(next < segments && keys[next < segments ? next * segment : 0] == key);
		if (inside == ~0ull) {
			parts += 64;
			continue;
		}
		parts += __builtin_ctzll(~inside);
		break;
	}
	for (size_t c0 = (size_t)blockIdx.y * 64 * VEC; c0 < cols; c0 += (size_t)gridDim.y * 64 * VEC) {
		const size_t c = c0 + (size_t)lane * VEC;
		Vec sum = Vec(0.0f);
		if (c < cols) {
			if (wave == 0) sum = *reinterpret_cast<const Vec*>(partial + ((size_t)s * 2 + 1) * cols + c);
			uint32_t q = wave;
			for (; q + 7 * kJoinWaves < parts; q += 8 * kJoinWaves) {
				Vec t[8];
#pragma unroll
				for (int u = 0; u < 8; u++) t[u] = *reinterpret_cast<const Vec*>(partial + ((size_t)s + 1 + q + u * kJoinWaves) * 2 * cols + c);
#pragma unroll
				for (int u = 0; u < 8; u++) sum += t[u];
			}
			for (; q < parts; q += kJoinWaves) sum += *reinterpret_cast<const Vec*>(partial + ((size_t)s + 1 + q) * 2 * cols + c);
		}
		sums[wave][lane] = sum;
		__syncthreads();
		if (wave == 0 && c < cols) {
#pragma unroll
			for (int w = 1; w < kJoinWaves; w++) sum += sums[w][lane];
			__builtin_nontemporal_store(sum * scale, reinterpret_cast<Vec*>(dtable + (size_t)key * cols + c));
		}
		__syncthreads();
	}
}

template <int VEC>
static int embedding_sums(const uint32_t* keys, const uint32_t* order, const float* dy, float* dtable, float* partial, uint32_t n, uint32_t vocab, size_t cols, float scale, uint32_t segment,
                          int lanes) {
	State& s = state();
	const uint32_t segments = (n + segment - 1) / segment;
	const size_t col_steps = (cols + (size_t)lanes * VEC - 1) / ((size_t)lanes * VEC);
	const size_t sum_groups = ((size_t)segments * col_steps * lanes + 255) / 256;
	size_t zero_groups = ((size_t)vocab + kZeroRows * 4 - 1) / (kZeroRows * 4);
	if (zero_groups > 1 << 20) zero_groups = 1 << 20;
	if (sum_groups + zero_groups > 0xFFFFFF) return fail(TFHIP_ERR_ARG, "embedding gradient of %u tokens with %zu columns is too large", n, cols);
	hipLaunchKernelGGL(embedding_sum_kernel<VEC>, dim3((unsigned)(sum_groups + zero_groups)), dim3(256), 0, s.stream, keys, order, dy, dtable, partial, n, vocab, cols, scale, segment, segments,
	                   lanes, (uint32_t)col_steps, (uint32_t)sum_groups);
	TFHIP_CHECK_LAUNCH();
	if (segments > 1) {
		const size_t stretches = (cols + 64 * VEC - 1) / (64 * VEC);
		hipLaunchKernelGGL(embedding_join_kernel<VEC>, dim3(segments - 1, (unsigned)(stretches < 16 ? stretches : 16)), dim3(kJoinWaves * 64), 0, s.stream, keys, dtable, (const float*)partial, n, vocab, cols, scale, segment, segments);
		TFHIP_CHECK_LAUNCH();
	}
	return TFHIP_OK;
}

// ---- few positions ----------------------------------------------------------------------------------------

// Up to kFewPositions positions in one launch, without an order of all of them. A group owns some rows of the table, the 64 VEC
// columns of a wave of them: it counts the positions of each, with the tokens in group memory, writes zeros into the rows
// without any as one stretch of memory, and adds up the others. A wave takes a row with few positions, which it finds in
// their order by a ballot for every 64 tokens; a row with more than kFewAlone is cut into eight parts of neighbouring positions, one
// per wave, added in their order at the end. us in the kernels, this one | the three launches below, which also wait for each
// other for 6 us in all: 500 x 250 over 1009 rows 5.8 | 14.0, 37 x 560 over 22709 11 | 21, 1000 x 1024 over 100 9.0 | 14.6, 1551 x 86
// over 6876 8.7 | 15.8, 2048 x 256 over 50000 13.6 | 24.9; and 4096 x 100 over 100 34 | 20.
// A group owns eight rows or more and goes through those with many positions one after the other, so the table needs rows enough
// to spread the positions: from kFewAnyTable positions on, one for kFewShare of them. us per call, tokens spread evenly:
//   2048 x 256 over 8 rows 47 | 16, 50 rows 31 | 16, 64 rows 24 | 16, 100 rows 8 | 16 (with a few frequent ones 16 | 16)
//   1024 x 256 over 8 rows 27 | 14, 32 rows 15 | 14, 64 rows 6 | 15;  512 x 256 over 8 rows 18 | 13, 16 rows 14 | 13;  256 x 256 over 8 rows 12 | 13
// (tables of one or two rows have no such queue and give up a little of it: 512 x 256 over one row 8 | 12, over two 10 | 12)
constexpr uint32_t kFewPositions = 2048, kFewMostRows = 256, kFewAnyTable = 384, kFewShare = 24;
constexpr int kFewWaves = 8, kFewThreads = kFewWaves * 64, kFewAlone = 32;
constexpr size_t kFewVocab = (size_t)1 << 30, kFewCols = 65535 * 64;  // a launch has fewer than 2^32 threads

template <int VEC>
__global__ __launch_bounds__(kFewThreads) void embedding_few_kernel(const int32_t* __restrict__ tokens, const float* __restrict__ dy, float* __restrict__ dtable, uint32_t n, uint32_t vocab,
                                                                    size_t cols, float scale, uint32_t rows_of_group) {
	typedef typename Floats<VEC>::type Vec;
	__shared__ uint32_t token[kFewPositions];
	__shared__ uint32_t count[kFewMostRows];
	__shared__ uint16_t list[kFewWaves][kFewAlone], long_list[kFewPositions];
	__shared__ Vec parts[kFewWaves][64];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const uint32_t v0 = blockIdx.x * rows_of_group, rows = vocab - v0 < rows_of_group ? vocab - v0 : rows_of_group;
	const size_t c = (size_t)blockIdx.y * 64 * VEC + (size_t)lane * VEC;  // this lane's columns
	const bool inside = c < cols;
	const uint32_t chunks = (n + 63) / 64;
	for (uint32_t r = threadIdx.x; r < kFewMostRows; r += kFewThreads) count[r] = 0;
	__syncthreads();
#pragma unroll
	for (uint32_t j = 0; j < kFewPositions / kFewThreads; j++) {
		const uint32_t i = j * kFewThreads + threadIdx.x;
		const uint32_t t = i < n ? (uint32_t)tokens[i] : 0xFFFFFFFFu;  // which names no row
		token[i] = t;
		if (t - v0 < rows) atomicAdd(&count[t - v0], 1u);
	}
	__syncthreads();
	const size_t c0 = (size_t)blockIdx.y * 64 * VEC;
	const uint32_t width = (uint32_t)(cols - c0 < 64 * VEC ? (cols - c0) / VEC : 64);
	for (uint32_t i = threadIdx.x; i < rows * width; i += kFewThreads) {
		const uint32_t r = i / width;
		if (count[r] == 0) __builtin_nontemporal_store(Vec(0.0f), reinterpret_cast<Vec*>(dtable + (size_t)(v0 + r) * cols + c0 + (i - r * width) * VEC));
	}
	// the sum of the rows of dy that `from` lists in [first, last)
	auto add_up = [&](const uint16_t* from, uint32_t first, uint32_t last) {
		Vec sum = Vec(0.0f);
		if (!inside) return sum;
		for (uint32_t p0 = first; p0 < last; p0 += kSumRows) {
			Vec v[kSumRows];
#pragma unroll
			for (int u = 0; u < kSumRows; u++) v[u] = *reinterpret_cast<const Vec*>(dy + (size_t)from[p0 + u < last ? p0 + u : p0] * cols + c);
#pragma unroll
			for (int u = 0; u < kSumRows; u++)
				if (p0 + u < last) sum += v[u];
		}
		return sum;
	};
	uint32_t turn = 0;  // rows with few positions go to the waves in turn
	for (uint32_t r0 = 0; r0 < rows; r0 += 64) {
		const uint32_t of_lane = count[r0 + lane];
		uint64_t few = __ballot(of_lane > 0 && of_lane <= kFewAlone);
		for (; few; few &= few - 1) {
			if (turn++ % kFewWaves != (uint32_t)wave) continue;
			const uint32_t r = r0 + __builtin_ctzll(few), found = count[r];
			uint32_t at = 0;
			for (uint32_t k = 0; k < chunks; k++) {
				const uint64_t same = __ballot(token[k * 64 + lane] == v0 + r);
				if ((same >> lane) & 1) list[wave][at + __popcll(same & ((1ull << lane) - 1))] = (uint16_t)(k * 64 + lane);
				at += __popcll(same);
			}
			__builtin_amdgcn_wave_barrier();
			const Vec sum = add_up(list[wave], 0, found);
			if (inside) __builtin_nontemporal_store(sum * scale, reinterpret_cast<Vec*>(dtable + (size_t)(v0 + r) * cols + c));
			__builtin_amdgcn_wave_barrier();
		}
	}
	for (uint32_t r0 = 0; r0 < rows; r0 += 64) {
		const uint32_t of_lane = count[r0 + lane];
		for (uint64_t many = __ballot(of_lane > kFewAlone); many; many &= many - 1) {  // the same in every wave
			const uint32_t r = r0 + __builtin_ctzll(many), found = count[r];
			uint32_t at = 0;
			for (uint32_t k = 0; k < chunks; k++) {
				const uint64_t same = __ballot(token[k * 64 + lane] == v0 + r);
				if (k % kFewWaves == (uint32_t)wave && ((same >> lane) & 1)) long_list[at + __popcll(same & ((1ull << lane) - 1))] = (uint16_t)(k * 64 + lane);
				at += __popcll(same);
			}
			__syncthreads();
			const uint32_t share = (found + kFewWaves - 1) / kFewWaves, first = wave * share < found ? wave * share : found, last = first + share < found ? first + share : found;
			Vec sum = add_up(long_list, first, last);
			parts[wave][lane] = sum;
			__syncthreads();
			if (wave == 0 && inside) {
#pragma unroll
				for (int w = 1; w < kFewWaves; w++) sum += parts[w][lane];
				__builtin_nontemporal_store(sum * scale, reinterpret_cast<Vec*>(dtable + (size_t)(v0 + r) * cols + c));
			}
			__syncthreads();
		}
	}
}

static int check_embedding(const char* what, size_t n, size_t vocab, size_t cols) {
	if (vocab == 0 || cols == 0) return fail(TFHIP_ERR_ARG, "%s with an empty table (%zu x %zu)", what, vocab, cols);
	if (n >= ((size_t)1 << 30)) return fail(TFHIP_ERR_ARG, "%s takes fewer than 2^30 tokens (got %zu)", what, n);
	if (vocab > 0x7FFFFFFF || cols > 0x7FFFFFFF) return fail(TFHIP_ERR_ARG, "%s with a table of %zu x %zu: a dimension is beyond 2^31 - 1", what, vocab, cols);
	return TFHIP_OK;
}

}  // namespace tfhip

using namespace tfhip;

extern "C" int tfhip_embedding_rows_f32(const int32_t* tokens, const float* table, float* out, size_t n, size_t vocab, size_t cols, float scale) {
	int rc = check_embedding("embedding lookup", n, vocab, cols);
	if (rc) return rc;
	if (n == 0) return TFHIP_OK;
	if (!tokens || !table || !out) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_embedding_rows_f32");
	if (words_overlap(out, n * cols, table, vocab * cols) || words_overlap(out, n * cols, tokens, n)) return fail(TFHIP_ERR_ARG, "embedding lookup: out overlaps the table or the tokens");
	TFHIP_REQUIRE_INIT();
	TFHIP_HOLD_DEVICE();
	State& s = state();
	const RowShape r = row_shape(cols, table, out);
	const size_t rows = (size_t)(256 / r.lanes) * kLookupRows, most = (size_t)s.compute_units * 32;
	size_t groups = (n + rows - 1) / rows;
	if (groups > most) groups = most;
	const dim3 grid((unsigned)groups), block(256);
	switch (r.vec) {
		case 4: hipLaunchKernelGGL(embedding_kernel<4>, grid, block, 0, s.stream, tokens, table, out, n, vocab, cols, scale, r.lanes); break;
		case 2: hipLaunchKernelGGL(embedding_kernel<2>, grid, block, 0, s.stream, tokens, table, out, n, vocab, cols, scale, r.lanes); break;
		default: hipLaunchKernelGGL(embedding_kernel<1>, grid, block, 0, s.stream, tokens, table, out, n, vocab, cols, scale, r.lanes); break;
	}
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}

extern "C" int tfhip_embedding_rows_backward_f32(const int32_t* tokens, const float* dy, float* dtable, size_t n, size_t vocab, size_t cols, float scale) {
	int rc = check_embedding("embedding gradient", n, vocab, cols);
	if (rc) return rc;
	if (!dtable || (n && (!tokens || !dy))) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_embedding_rows_backward_f32");
	if (words_overlap(dtable, vocab * cols, dy, n * cols) || words_overlap(dtable, vocab * cols, tokens, n))
		return fail(TFHIP_ERR_ARG, "embedding gradient: dtable overlaps dy or the tokens");
	TFHIP_REQUIRE_INIT();
	TFHIP_HOLD_DEVICE();
	State& s = state();
	if (n == 0) return tfhip_fill_u32(dtable, 0u, vocab * cols);
	if (n <= kFewPositions && (n <= kFewAnyTable || n <= vocab * kFewShare) && vocab <= kFewVocab && cols <= kFewCols) {
		const RowShape r = row_shape(cols, dy, dtable);
		// four groups a unit, with 8 to kFewMostRows rows each
		const size_t stretches = (cols + 64 * r.vec - 1) / (64 * r.vec), wanted = (vocab * stretches + s.compute_units * 4 - 1) / (s.compute_units * 4);
		const size_t rows = wanted < 8 ? 8 : wanted < kFewMostRows ? wanted : kFewMostRows;
		const dim3 grid((unsigned)((vocab + rows - 1) / rows), (unsigned)stretches), block(kFewThreads);
		switch (r.vec) {
			case 4: hipLaunchKernelGGL(embedding_few_kernel<4>, grid, block, 0, s.stream, tokens, dy, dtable, (uint32_t)n, (uint32_t)vocab, cols, scale, (uint32_t)rows); break;
			case 2: hipLaunchKernelGGL(embedding_few_kernel<2>, grid, block, 0, s.stream, tokens, dy, dtable, (uint32_t)n, (uint32_t)vocab, cols, scale, (uint32_t)rows); break;
			default: hipLaunchKernelGGL(embedding_few_kernel<1>, grid, block, 0, s.stream, tokens, dy, dtable, (uint32_t)n, (uint32_t)vocab, cols, scale, (uint32_t)rows); break;
		}
		TFHIP_CHECK_LAUNCH();
		return TFHIP_OK;
	}
	const bool radix = n > kMostTiled;
	int digits = 1;  // of keys 0 .. vocab
	while (digits < 4 && vocab >> (8 * digits)) digits++;
	// Rows a wave adds up one after the other: few rows need shorter chains, more of them at once (sums and joins, us, with 16 | 32:
	// 4096 x 512 9.6 | 11.7, 8192 x 64 10.2 | 12.1), many rows fewer parts to join (65536 x 1024 93 | 89, with 64 88.5).
	uint32_t segment = n * cols >= (size_t)1 << 22 ? 32 : 16;
	while (n / segment >= (size_t)1 << 22) segment *= 2;  // a launch has fewer than 2^32 threads
	const size_t segments = (n + segment - 1) / segment;
	// [the library sort's own words][keys, order sorted][keys, order between passes, and before them][counts][parts of the runs]
	const size_t words = (n + 63) & ~size_t(63);
	const uint32_t tiles = (uint32_t)((n + kDigitTile - 1) / kDigitTile);
	const size_t sort_bytes = radix ? radix_sort_scratch_bytes(n) : 0, arrays = n <= kAllPairs ? 2 : radix ? 6 : 4;
	const size_t count_words = radix || n <= kAllPairs ? 0 : (size_t)tiles * 256;
	char* base = (char*)scratch(sort_bytes + (arrays * words + count_words) * sizeof(uint32_t) + segments * 2 * cols * sizeof(float));
	if (!base) return TFHIP_ERR_HIP;
	uint32_t* keys = (uint32_t*)(base + sort_bytes);
	uint32_t* order = keys + words;
	uint32_t* counts = keys + arrays * words;
	float* partial = (float*)(counts + count_words);
	if (radix) {
		hipLaunchKernelGGL(embedding_keys_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s.stream, tokens, keys + 2 * words, keys + 3 * words, (uint32_t)n, (uint32_t)vocab);
		TFHIP_CHECK_LAUNCH();
		rc = radix_sort_low_digits(keys + 2 * words, keys + 3 * words, keys, order, keys + 4 * words, keys + 5 * words, n, digits);
		if (rc) return rc;
	} else if (n > kAllPairs) {
		for (int p = 0; p < digits; p++) {
			// the last pass ends in keys and order
			const bool away = (digits - 1 - p) & 1;
			const uint32_t* from = away ? keys : keys + 2 * words;
			uint32_t* to = away ? keys + 2 * words : keys;
			const dim3 grid(tiles), block(256);
			if (p == 0) {
				hipLaunchKernelGGL(embedding_digits_kernel<true>, grid, block, 0, s.stream, tokens, from, counts, (uint32_t)n, (uint32_t)vocab, 0);
				TFHIP_CHECK_LAUNCH();
				hipLaunchKernelGGL(embedding_scatter_kernel<true>, grid, block, 0, s.stream, tokens, from, from + words, to, to + words, (const uint32_t*)counts, (uint32_t)n, (uint32_t)vocab, tiles, 0);
			} else {
				hipLaunchKernelGGL(embedding_digits_kernel<false>, grid, block, 0, s.stream, tokens, from, counts, (uint32_t)n, (uint32_t)vocab, 8 * p);
				TFHIP_CHECK_LAUNCH();
				hipLaunchKernelGGL(embedding_scatter_kernel<false>, grid, block, 0, s.stream, tokens, from, from + words, to, to + words, (const uint32_t*)counts, (uint32_t)n, (uint32_t)vocab, tiles,
				                   8 * p);
			}
			TFHIP_CHECK_LAUNCH();
		}
	} else {
		hipLaunchKernelGGL(embedding_count_kernel, dim3((unsigned)((n + 63) / 64)), dim3(kCountWaves * 64), 0, s.stream, (const uint32_t*)tokens, keys, order, (uint32_t)n);
		TFHIP_CHECK_LAUNCH();
	}
	const RowShape r = row_shape(cols, dy, dtable);
	switch (r.vec) {
		case 4: return embedding_sums<4>(keys, order, dy, dtable, partial, (uint32_t)n, (uint32_t)vocab, cols, scale, segment, r.lanes);
		case 2: return embedding_sums<2>(keys, order, dy, dtable, partial, (uint32_t)n, (uint32_t)vocab, cols, scale, segment, r.lanes);
		default: return embedding_sums<1>(keys, order, dy, dtable, partial, (uint32_t)n, (uint32_t)vocab, cols, scale, segment, r.lanes);
	}
}
