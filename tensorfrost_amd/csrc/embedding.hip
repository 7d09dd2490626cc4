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

// A position's key is its token, or vocab where the token names no row. The sorted keys and positions of a tile come
// from counting: the place of position i is the number of keys that are smaller, or equal and earlier. A group places 64
// positions; its four waves each compare them with a quarter of the tile's keys, a compare and an add per pair:
// tile * 64 pairs take about 2 tile cycles. Up to kAllPairs positions are one tile; beyond, tiles of kSortTile are sorted
// so and merged by searches.
constexpr uint32_t kAllPairs = 8192, kSortTile = 1024, kMostSearched = 131072;

__device__ __forceinline__ uint32_t token_key(int32_t t, uint32_t vocab) { return t >= 0 && (uint32_t)t < vocab ? (uint32_t)t : vocab; }

__global__ __launch_bounds__(256) void embedding_count_kernel(const int32_t* __restrict__ tokens, uint32_t* __restrict__ keys, uint32_t* __restrict__ order, uint32_t n, uint32_t vocab,
                                                              uint32_t tile) {
	__shared__ __attribute__((aligned(16))) uint32_t key[kAllPairs];
	__shared__ uint32_t counts[4][64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const uint32_t first = blockIdx.x * 64 / tile * tile;              // the tile's first position
	const uint32_t count = n - first < tile ? n - first : tile;
	const uint32_t blocks = (count + 63) / 64;
	for (uint32_t i = threadIdx.x; i < blocks * 64; i += 256) key[i] = i < count ? token_key(tokens[first + i], vocab) : 0xFFFFFFFFu;
	__syncthreads();
	const uint32_t mine = blockIdx.x * 64 - first + lane, my_block = mine / 64;
	const uint32_t k = key[mine];
	uint32_t before = 0;
	for (uint32_t b = wave; b < blocks; b += 4) {
		const uint4* other = reinterpret_cast<const uint4*>(key + b * 64);
		if (b != my_block) {
			const uint32_t below = b < my_block ? k + 1 : k;  // equal keys count when they stand before
#pragma unroll
			for (int j = 0; j < 16; j++) {
				const uint4 o = other[j];
				before += (o.x < below) + (o.y < below) + (o.z < below) + (o.w < below);
			}
		} else {
			for (int j = 0; j < 64; j++) before += key[b * 64 + j] < k + (j < lane);
		}
	}
	counts[wave][lane] = before;
	__syncthreads();
	if (wave == 0 && mine < count) {
		const uint32_t at = first + counts[0][lane] + counts[1][lane] + counts[2][lane] + counts[3][lane];
		keys[at] = k;
		order[at] = first + mine;
	}
}

// Merges sorted tiles of kSortTile: the place of an element is its place in its own tile plus, for every other tile, the
// number of that tile's keys that come before it (binary search in group memory; tiles before count equal keys, tiles
// behind do not). A group places 256 elements; four threads share an element and search a tile each of the four
// that a thread group has in flight. The last tile may be short: it is filled up with the largest key.
constexpr int kMergeTiles = 16;
__global__ __launch_bounds__(1024) void embedding_merge_kernel(const uint32_t* __restrict__ tile_keys, const uint32_t* __restrict__ tile_order, uint32_t* __restrict__ keys,
                                                               uint32_t* __restrict__ order, uint32_t n) {
	__shared__ uint32_t lds[kMergeTiles * kSortTile];
	__shared__ uint32_t counts[4][256];
	const uint32_t item = threadIdx.x & 255, quarter = threadIdx.x >> 8;
	const uint32_t e = blockIdx.x * 256 + item, tile = blockIdx.x * 256 / kSortTile, tiles = (n + kSortTile - 1) / kSortTile;
	const uint32_t k = e < n ? tile_keys[e] : 0xFFFFFFFEu;
	uint32_t before = 0;
	for (uint32_t t0 = 0; t0 < tiles; t0 += kMergeTiles) {
		__syncthreads();
#pragma unroll
		for (int i = 0; i < kMergeTiles; i++) {
			const uint32_t at = (t0 + i) * kSortTile + threadIdx.x;
			lds[i * kSortTile + threadIdx.x] = at < n ? tile_keys[at] : 0xFFFFFFFFu;
		}
		__syncthreads();
		uint32_t found[4] = {0, 0, 0, 0}, below[4];
#pragma unroll
		for (int i = 0; i < 4; i++) below[i] = t0 + quarter * 4 + i < tile ? k + 1 : k;
#pragma unroll
		for (uint32_t half = kSortTile / 2; half >= 1; half /= 2)
#pragma unroll
			for (int i = 0; i < 4; i++) found[i] += lds[(quarter * 4 + i) * kSortTile + found[i] + half - 1] < below[i] ? half : 0;
#pragma unroll
		for (int i = 0; i < 4; i++) {
			found[i] += lds[(quarter * 4 + i) * kSortTile + found[i]] < below[i];  // found <= kSortTile - 1 here
			if (t0 + quarter * 4 + i != tile) before += found[i];
		}
	}
	counts[quarter][item] = before;
	__syncthreads();
	if (quarter == 0 && e < n) {
		const uint32_t at = e - tile * kSortTile + counts[0][item] + counts[1][item] + counts[2][item] + counts[3][item];
		keys[at] = k;
		order[at] = tile_order[e];
	}
}

// For the radix sort: keys[i] as above, order[i] = i.
__global__ __launch_bounds__(256) void embedding_keys_kernel(const int32_t* __restrict__ tokens, uint32_t* __restrict__ keys, uint32_t* __restrict__ order, uint32_t n, uint32_t vocab) {
	const uint32_t i = blockIdx.x * 256 + threadIdx.x;
	if (i >= n) return;
	keys[i] = token_key(tokens[i], vocab);
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
// The groups behind those of the segments write zeros into the rows that no position names, kZeroRows rows a wave:
// whether a row is named is found by a search for it, all rows of a wave at once.
constexpr int kSumRows = 8, kZeroRows = 16;

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
		for (uint32_t p0 = begin; p0 < end; p0 += kSumRows) {
			uint32_t k[kSumRows];
			size_t row[kSumRows];
			Vec v[kSumRows];
#pragma unroll
			for (int u = 0; u < kSumRows; u++) {
				const uint32_t p = p0 + u < end ? p0 + u : end - 1;
				k[u] = keys[p];
				row[u] = (size_t)order[p] * cols;
			}
#pragma unroll
			for (int u = 0; u < kSumRows; u++) v[u] = __builtin_nontemporal_load(reinterpret_cast<const Vec*>(dy + row[u] + c));
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
	const uint32_t v0 = ((blockIdx.x - sum_groups) * 4 + (threadIdx.x >> 6)) * kZeroRows;
	if (v0 >= vocab) return;
	bool idle = false;
	if (lane < kZeroRows && v0 + lane < vocab) {
		const uint32_t at = first_at_least(keys, n, v0 + lane);
		idle = at >= n || keys[at] != v0 + lane;
	}
	uint64_t rows = __ballot(idle);
	while (rows) {
		const int r = __builtin_ctzll(rows);
		rows &= rows - 1;
		float* to = dtable + (size_t)(v0 + r) * cols;
		for (size_t c = (size_t)lane * VEC; c < cols; c += 64 * VEC) __builtin_nontemporal_store(Vec(0.0f), reinterpret_cast<Vec*>(to + c));
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
	for (size_t c0 = 0; c0 < cols; c0 += 64 * VEC) {
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
	const size_t sum_groups = ((size_t)segments * col_steps * lanes + 255) / 256, zero_groups = ((size_t)vocab + kZeroRows * 4 - 1) / (kZeroRows * 4);
	if (sum_groups + zero_groups > 0x7FFFFFFF) return fail(TFHIP_ERR_ARG, "embedding gradient of %u tokens with %zu columns is too large", n, cols);
	hipLaunchKernelGGL(embedding_sum_kernel<VEC>, dim3((unsigned)(sum_groups + zero_groups)), dim3(256), 0, s.stream, keys, order, dy, dtable, partial, n, vocab, cols, scale, segment, segments,
	                   lanes, (uint32_t)col_steps, (uint32_t)sum_groups);
	TFHIP_CHECK_LAUNCH();
	if (segments > 1) {
		hipLaunchKernelGGL(embedding_join_kernel<VEC>, dim3(segments - 1), dim3(kJoinWaves * 64), 0, s.stream, keys, dtable, (const float*)partial, n, vocab, cols, scale, segment, segments);
		TFHIP_CHECK_LAUNCH();
	}
	return TFHIP_OK;
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
	const bool radix = n > kMostSearched;
	const uint32_t segment = n * cols >= (size_t)1 << 22 ? 64 : 16;  // few rows: shorter chains of loads, more of them at once
	const size_t segments = (n + segment - 1) / segment;
	// [the sort's own words][keys, order sorted][keys, order before (and between) the sort's passes][parts of the runs]
	const size_t words = (n + 63) & ~size_t(63);
	const size_t sort_bytes = radix ? radix_sort_scratch_bytes(n) : 0, arrays = n <= kAllPairs ? 2 : radix ? 6 : 4;
	char* base = (char*)scratch(sort_bytes + arrays * words * sizeof(uint32_t) + segments * 2 * cols * sizeof(float));
	if (!base) return TFHIP_ERR_HIP;
	uint32_t* keys = (uint32_t*)(base + sort_bytes);
	uint32_t* order = keys + words;
	float* partial = (float*)(keys + arrays * words);
	if (radix) {
		hipLaunchKernelGGL(embedding_keys_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s.stream, tokens, keys + 2 * words, keys + 3 * words, (uint32_t)n, (uint32_t)vocab);
		TFHIP_CHECK_LAUNCH();
		rc = tfhip_radix_sort_kv_u32(keys + 2 * words, keys + 3 * words, keys, order, keys + 4 * words, keys + 5 * words, n);
		if (rc) return rc;
	} else if (n > kAllPairs) {
		hipLaunchKernelGGL(embedding_count_kernel, dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s.stream, tokens, keys + 2 * words, keys + 3 * words, (uint32_t)n, (uint32_t)vocab, kSortTile);
		TFHIP_CHECK_LAUNCH();
		hipLaunchKernelGGL(embedding_merge_kernel, dim3((unsigned)((n + 255) / 256)), dim3(1024), 0, s.stream, (const uint32_t*)(keys + 2 * words), (const uint32_t*)(keys + 3 * words), keys, order,
		                   (uint32_t)n);
		TFHIP_CHECK_LAUNCH();
	} else {
		hipLaunchKernelGGL(embedding_count_kernel, dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s.stream, tokens, keys, order, (uint32_t)n, (uint32_t)vocab, kAllPairs);
		TFHIP_CHECK_LAUNCH();
	}
	const RowShape r = row_shape(cols, dy, dtable);
	switch (r.vec) {
		case 4: return embedding_sums<4>(keys, order, dy, dtable, partial, (uint32_t)n, (uint32_t)vocab, cols, scale, segment, r.lanes);
		case 2: return embedding_sums<2>(keys, order, dy, dtable, partial, (uint32_t)n, (uint32_t)vocab, cols, scale, segment, r.lanes);
		default: return embedding_sums<1>(keys, order, dy, dtable, partial, (uint32_t)n, (uint32_t)vocab, cols, scale, segment, r.lanes);
	}
}
