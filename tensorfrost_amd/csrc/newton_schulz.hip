// Orthogonalisation of matrices by Newton-Schulz products, as optimisers apply it to the update of a dense layer:
//
//   X = G / (|G|_F + eps);  per step, with its coefficients a, b, c:  A = X X^T,  B = b A + c A^2,  X <- a X + B X
//
// (on the transposed matrix when there are more rows than columns, so that A is the smaller of the two squares). Each
// singular value s of X becomes a s + b s^3 + c s^5. The reference has no such operation; its optimisers stop at the
// element-wise update (Python/TensorFrost/optimizers.py:104-167).
//
// Number format. The fp32 matrix instructions reach 157 TFLOP/s here, the fp16 ones 2500. So every operand is held as a
// pair of fp16 numbers in 32 bits, v = (hi + lo) / scale with hi = fp16(v scale), lo = fp16(v scale - hi), and a product is
// three fp16 products into one fp32 accumulator, hi hi + hi lo + lo hi. The pair keeps 22 bits, one less than fp32 keeps
// on average, and the dropped lo lo is below 2^-22 of the product; in exchange the accumulator takes 16 terms a step instead of
// 2, and the result after five steps is as far from the 64-bit one as that of fp32 products (1.3e-6 against 1.6e-6 of the norm at
// 256 x 256). The scale is a power of two from a bound on the spectral norm, which no element exceeds: of X it is 1 at the start (or, for a
// G below eps, the power of two above |X|) and after a step max |a s + b s^3 + c s^5| over the reachable s; the scale puts that bound
// between 2^14 and 2^15. hi is off by at most 2^-11 of the power of two below v, lo holds that to 2^-12 of itself, so the pair is
// within 2^-23 of v, until lo reaches the fixed grid of 2^-24 of small fp16 numbers: elements below 2^-16 of the bound keep an
// absolute error of 2^-39 of it instead.
//
// Layout. A row of a split matrix is a sequence of 128-byte blocks, 32 hi then the 32 lo of the same columns, so one
// cache line holds a row's share of a step of 32 in k. Rows and columns are padded to whole tiles with zeros, which stay
// zeros through every product: no kernel but the first and the last tests a bound. All products have both operands
// contiguous along k (row i of P times row j of Q): A and B are symmetric, and X is kept in both orientations.

#include "common.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace tfhip {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

constexpr int kNsBlock = 128;  // bytes of a row's block: 32 columns, hi and lo
constexpr int kNsStep = 32;    // columns of a block

// ---- split values --------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t split_pair(float v) {
	const _Float16 hi = (_Float16)v;
	const _Float16 lo = (_Float16)(v - (float)hi);
	return (uint32_t)__builtin_bit_cast(unsigned short, hi) | ((uint32_t)__builtin_bit_cast(unsigned short, lo) << 16);
}

// One wave writes a 32 x 32 tile of split values that its lanes hold in the layout of a 32 x 32 accumulator (element r of
// lane l: row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32) as 32 whole blocks: `straight` receives rows (block i =
// row i), `turned` columns (block i = column i); either may be null. `lds` is 32 x 33 words of this wave's own.
__device__ __forceinline__ void store_split_tile(const float (&v)[16], uint32_t* lds, char* straight, size_t straight_stride, char* turned, size_t turned_stride) {
	const int lane = threadIdx.x & 63;
	__builtin_amdgcn_wave_barrier();
#pragma unroll
	for (int r = 0; r < 16; r++) lds[(8 * (r / 4) + 4 * (lane >> 5) + r % 4) * 33 + (lane & 31)] = split_pair(v[r]);
	__builtin_amdgcn_wave_barrier();
	const int line = lane >> 1, part = lane & 1;  // two lanes a block: 16 of its columns each
#pragma unroll
	for (int form = 0; form < 2; form++) {
		char* to = form == 0 ? straight : turned;
		if (!to) continue;
		uint32_t hi[8], lo[8];
#pragma unroll
		for (int k = 0; k < 8; k++) {
			const int c = part * 16 + 2 * k;
			const uint32_t p = form == 0 ? lds[line * 33 + c] : lds[c * 33 + line];
			const uint32_t q = form == 0 ? lds[line * 33 + c + 1] : lds[(c + 1) * 33 + line];
			hi[k] = (p & 0xFFFFu) | (q << 16);
			lo[k] = (p >> 16) | (q & 0xFFFF0000u);
		}
		char* at = to + (size_t)line * (form == 0 ? straight_stride : turned_stride) + part * 32;
		*reinterpret_cast<uintx4*>(at) = uintx4{hi[0], hi[1], hi[2], hi[3]};
		*reinterpret_cast<uintx4*>(at + 16) = uintx4{hi[4], hi[5], hi[6], hi[7]};
		*reinterpret_cast<uintx4*>(at + 64) = uintx4{lo[0], lo[1], lo[2], lo[3]};
		*reinterpret_cast<uintx4*>(at + 80) = uintx4{lo[4], lo[5], lo[6], lo[7]};
	}
}

// ---- scales --------------------------------------------------------------------------------------

// max |a s + b s^3 + c s^5| over s in [0, top]: at the end or where the derivative is 0.
__host__ __device__ inline double largest_quintic(double a, double b, double c, double top) {
	double best = 0.0;
	auto look = [&](double t) {  // t = s^2
		if (!(t >= 0.0 && t <= top * top)) return;
		const double p = fabs((a + t * (b + t * c)) * sqrt(t));
		if (!(p <= best)) best = p;
	};
	look(top * top);
	const double u = a, v = 3.0 * b, w = 5.0 * c;  // u + v t + w t^2 = 0
	if (w == 0.0) {
		if (v != 0.0) look(-u / v);
	} else if (v * v - 4.0 * u * w >= 0.0) {
		const double root = sqrt(v * v - 4.0 * u * w);
		look((-v + root) / (2.0 * w));
		look((-v - root) / (2.0 * w));
	}
	return best;
}

// max |b t + c t^2| over t in [0, top], likewise.
__host__ __device__ inline double largest_square(double b, double c, double top) {
	const double end = fabs(top * (b + top * c)), t = c != 0.0 ? -b / (2.0 * c) : -1.0;
	const double middle = t > 0.0 && t < top ? fabs(t * (b + t * c)) : 0.0;
	return end > middle ? end : middle;
}

// The power of two that brings values of at most `bound` to at most 2^15.
__host__ __device__ inline double scale_for(double bound) {
	if (!(bound > 1e-30)) bound = 1e-30;
	if (!(bound < 1e37)) bound = 1e37;
	int e;
	frexp(bound, &e);  // bound <= 2^e
	return ldexp(1.0, 15 - e);
}

// What the products of a step are multiplied with on their way from one scale to another.
struct NsFactors {
	float gram;            // X X^T in A
	float poly, poly_a;    // A^2 and A in B
	float update, update_x;  // B X and X in the next X
};

// The scales of the split matrices, step by step.
struct NsScales {
	double bound;  // on the spectral norm of X
	double next;   // the scale of X
	__host__ __device__ explicit NsScales(double first) : bound(first), next(scale_for(first)) {}
	__host__ __device__ NsFactors step(const float* abc, bool last) {
		const double ca = abc[0], cb = abc[1], cc = abc[2], x = next;
		// bounds that rounding does not cross
		const double a = scale_for(bound * bound * 1.0001), b = scale_for(largest_square(cb, cc, bound * bound) * 1.0001);
		bound = largest_quintic(ca, cb, cc, bound) * 1.0001;
		next = last ? 1.0 : scale_for(bound);
		return {(float)(a / (x * x)), (float)(cc * b / (a * a)), (float)(cb * b / a), (float)(next / (b * x)), (float)(ca * next / x)};
	}
};

// The steps of a call: their coefficients, and their factors where |X| may be anything up to 1 at the start.
struct NsSteps {
	int count;
	float coefficients[64][3];
	NsFactors usual[64];
};

// What |X| = norm / (norm + eps) does not exceed: 1, or, where it is below a half, the next power of two, so that a gradient far below
// eps keeps the digits of its small X. (|G| = 1e-13 with eps = 1e-7, 1000 x 1020, five steps: the result is off by 1.2e-7, with a bound
// of 1 for all it was 1.1e-3.) Such a matrix has factors of its own, worked out by one thread of its group. The others pay for
// factors in memory: 2 of 256 x 256 80.9 -> 81.5 us, 512 x 512 102.9 -> 104.1, 64 x 256 in one group 40.3 -> 40.8.
__device__ inline double ns_first_bound(double norm, double eps) {
	if (!(norm < eps)) return 1.0;
	int e;
	frexp(norm / (norm + eps), &e);
	return ldexp(1.0, e);
}
__device__ inline void ns_own_factors(const NsSteps& steps, double first, NsFactors* to) {
	NsScales scales(first);
	for (int k = 0; k < steps.count; k++) to[k] = scales.step(steps.coefficients[k], k + 1 == steps.count);
}

// ---- the norm and the first split -----------------------------------------------------------------

// Partial sums of squares, in 64 bits: the square of a large fp32 number does not fit fp32. `vec`: every matrix starts on
// 16 bytes and holds whole vectors. (4096 x 4096, 64 MiB: 14 us, 4.7 TB/s; the split behind it, which writes both
// orientations, 42 us.)
__global__ __launch_bounds__(256) void ns_norm_kernel(const float* __restrict__ g, double* __restrict__ partial, size_t elements, unsigned parts, bool vec) {
	__shared__ double red[4];
	const size_t matrix = blockIdx.x / parts, part = blockIdx.x % parts;
	const float* p = g + matrix * elements;
	double sum = 0.0, sum2 = 0.0;
	if (vec) {
		const size_t vecs = elements / 4, step = (size_t)parts * 256;
		const float4* v = reinterpret_cast<const float4*>(p);
		size_t i = part * 256 + threadIdx.x;
		for (; i + 3 * step < vecs; i += 4 * step) {
			float4 t[4];
#pragma unroll
			for (int u = 0; u < 4; u++) t[u] = v[i + u * step];
#pragma unroll
			for (int u = 0; u < 4; u++) {
				sum += (double)t[u].x * (double)t[u].x + (double)t[u].y * (double)t[u].y;
				sum2 += (double)t[u].z * (double)t[u].z + (double)t[u].w * (double)t[u].w;
			}
		}
		for (; i < vecs; i += step) {
			const float4 t = v[i];
			sum += (double)t.x * (double)t.x + (double)t.y * (double)t.y;
			sum2 += (double)t.z * (double)t.z + (double)t.w * (double)t.w;
		}
	} else {
		for (size_t i = part * 256 + threadIdx.x; i < elements; i += (size_t)parts * 256) sum += (double)p[i] * (double)p[i];
	}
	sum = wave_reduce(sum + sum2, [](double a, double b) { return a + b; });
	if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
	__syncthreads();
	if (threadIdx.x == 0) partial[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// X and its transpose in split form from g. X is [mp, np] with mp, np padded; `transposed`: g is [n, m], else [m, n].
// A wave per 32 x 32 tile, taken in turn; each group adds up the norm's parts for itself once. The first group of a matrix writes
// its factors, [matrix][step].
__global__ __launch_bounds__(256) void ns_split_kernel(const float* __restrict__ g, const double* __restrict__ partial, unsigned parts, char* x, char* xt, size_t m, size_t n, size_t mp, size_t np,
                                                       bool transposed, float eps, NsFactors* __restrict__ factors, const NsSteps steps) {
	__shared__ uint32_t lds[4][32 * 33];
	__shared__ double red[4];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const size_t matrix = blockIdx.y, tiles_n = np / 32, tiles = tiles_n * (mp / 32), step = (size_t)gridDim.x * 4;
	// tiles in the orientation of g, so that its rows are read along memory
	const size_t rows = transposed ? n : m, cols = transposed ? m : n;
	g += matrix * m * n;
	float v[16];
	auto load = [&](size_t tile) {
		const size_t t0 = tile / tiles_n * 32, t1 = tile % tiles_n * 32, r0 = transposed ? t1 : t0, c0 = transposed ? t0 : t1;
#pragma unroll
		for (int k = 0; k < 16; k++) {
			const size_t row = r0 + 8 * (k / 4) + 4 * (lane >> 5) + k % 4, col = c0 + (lane & 31);
			v[k] = row < rows && col < cols ? g[row * cols + col] : 0.0f;
		}
	};
	size_t tile = (size_t)blockIdx.x * 4 + wave;
	if (tile < tiles) load(tile);
	double sum = 0.0;
	for (unsigned k = threadIdx.x; k < parts; k += 256) sum += partial[matrix * parts + k];
	sum = wave_reduce(sum, [](double a, double b) { return a + b; });
	if (lane == 0) red[wave] = sum;
	__syncthreads();
	const double own = sqrt((red[0] + red[1]) + (red[2] + red[3])), norm = own + (double)eps, first = ns_first_bound(own, eps);
	const double r = !isfinite(norm) ? (double)nanf("") : norm > 0.0 ? scale_for(first) / norm : 0.0;
	if (blockIdx.x == 0) {
		factors += matrix * steps.count;
		if (first == 1.0) {
			if ((int)threadIdx.x < steps.count) factors[threadIdx.x] = steps.usual[threadIdx.x];
		} else if (threadIdx.x == 0) {
			ns_own_factors(steps, first, factors);
		}
	}
	while (tile < tiles) {
		const size_t t0 = tile / tiles_n * 32, t1 = tile % tiles_n * 32;
#pragma unroll
		for (int k = 0; k < 16; k++) v[k] = (float)((double)v[k] * r);
		char* to_x = x + matrix * mp * np * 4 + t0 * np * 4 + t1 * 4;
		char* to_xt = xt + matrix * mp * np * 4 + t1 * mp * 4 + t0 * 4;
		store_split_tile(v, lds[wave], transposed ? to_xt : to_x, transposed ? mp * 4 : np * 4, transposed ? to_x : to_xt, transposed ? np * 4 : mp * 4);
		tile += step;
		if (tile < tiles) load(tile);
	}
}

// ---- the products ---------------------------------------------------------------------------------

enum NsKind {
	kNsGram,    // A = X X^T: tiles on and below the diagonal, each written in both orientations
	kNsPoly,    // B = b A + c A^2: the same tiles
	kNsUpdate,  // X <- a X + B X, written in both orientations
	kNsLast     // the same in fp32, into the caller's matrix
};

struct NsArgs {
	const char* P;  // tile rows: [p_tiles * TILE, k_blocks * 32]
	const char* Q;  // tile columns
	const char* addend;  // all but kNsGram: a matrix to add, as [row of Q, row of P]
	char* straight;  // out[row of P, row of Q]
	char* turned;    // out[row of Q, row of P]
	float* out;      // kNsLast: [out_rows, out_cols]
	size_t batch_p, batch_q, batch_addend, batch_out;          // bytes between the matrices of a batch
	size_t addend_stride, straight_stride, turned_stride;      // bytes between rows
	size_t out_rows, out_cols;
	uint32_t k_blocks;          // blocks of a row of P and Q
	uint32_t tiles_p, tiles_q;
	uint32_t band;  // tile rows of a patch
	uint32_t whole;   // tiles that one group each works on; the others are cut along k
	uint32_t cuts;    // into so many parts
	float4* partial;  // the parts' sums
	const NsFactors* factors;  // of this step of the first matrix
	uint32_t steps;            // of a matrix
};

// What an element of the accumulator is multiplied with, and one of the addend. Read at the start of a kernel, where nothing waits for it.
struct NsPair {
	float alpha, beta;
};
template <int KIND>
__device__ __forceinline__ NsPair pair_of(const NsArgs& g) {
	const NsFactors* f = g.factors + (size_t)blockIdx.y * g.steps;
	if (KIND == kNsGram) return {f->gram, 0.0f};
	if (KIND == kNsPoly) return {f->poly, f->poly_a};
	return {f->update, f->update_x};
}

__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p; }

// 16 bytes per lane from base + offset to group memory at `to` + 16 lane. No vector register is written; the data is there
// after a wait for the vector-memory counter. (m0 is set where it is used: nothing else in these kernels reads it.)
__device__ __forceinline__ void load_to_lds(uint32_t to, uint32_t offset, const char* base) {
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base) : "memory");
}

template <int LEFT>
__device__ __forceinline__ void wait_loads() {
	static_assert(LEFT >= 0 && LEFT < 64, "the counter has six bits");
	asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
}

// Which tile of the result a group works on. Consecutive groups go to different dies, each with its own L2: die d gets the
// d-th run of tiles, and a run fills a compact patch of the result (bands of `band` tile rows, walked down each column of
// the band before the next), so that a die reads as few different rows of P and Q as its share of the work allows.
// The symmetric products list each pair of tile rows once as (r, r + c modulo n), c = 0 .. n / 2 (for even n only half of
// the r at c = n / 2), which makes the triangle a rectangle of n rows.
// The tiles that are cut follow the whole ones.
__device__ __forceinline__ uint32_t whole_tile_of_group(const NsArgs& g) {
	const uint32_t q = g.whole >> 3, rem = g.whole & 7, die = blockIdx.x & 7;
	return die * q + (die < rem ? die : rem) + (blockIdx.x >> 3);
}
template <int KIND>
__device__ __forceinline__ void place_of_tile(const NsArgs& g, uint32_t t, uint32_t& tp, uint32_t& tq) {
	constexpr bool kHalf = KIND == kNsGram || KIND == kNsPoly;
	const uint32_t rows = g.tiles_p, cols = kHalf ? (g.tiles_p + 1) / 2 : g.tiles_q;
	uint32_t r, c;
	if (!kHalf || t < rows * cols) {
		const uint32_t top = t / (g.band * cols) * g.band, height = rows - top < g.band ? rows - top : g.band, at = t - top * cols;
		c = at / height;
		r = top + at - c * height;
	} else {
		c = cols;
		r = t - rows * cols;
	}
	if (kHalf) {
		c = r + c < rows ? r + c : r + c - rows;
		tp = r > c ? r : c;
		tq = r > c ? c : r;
	} else {
		tp = r;
		tq = c;
	}
}

// The 32 x 32 tile of the addend at (row0, col0) of the result. It is stored turned, so that the four rows of a lane are
// four neighbours in memory.
struct Addend {
	half4 hi[4], lo[4];
};
__device__ __forceinline__ void load_addend(const NsArgs& g, Addend& a, uint32_t row0, uint32_t col0) {
	const int lane = threadIdx.x & 63;
	const char* p = g.addend + blockIdx.y * g.batch_addend + (size_t)(col0 + (lane & 31)) * g.addend_stride + (size_t)row0 * 4 + 8 * (lane >> 5);
#pragma unroll
	for (int q = 0; q < 4; q++) {
		a.hi[q] = *reinterpret_cast<const half4*>(p + 16 * q);
		a.lo[q] = *reinterpret_cast<const half4*>(p + 16 * q + 64);
	}
}

// What a kind does with a finished 32 x 32 tile of P Q^T at (row0, col0), held by one wave in accumulator layout.
template <int KIND>
__device__ __forceinline__ void finish_tile(const NsArgs& g, const NsPair& by, float (&v)[16], const Addend& a, uint32_t row0, uint32_t col0, bool diagonal, uint32_t* corner) {
	const int lane = threadIdx.x & 63;
#pragma unroll
	for (int r = 0; r < 16; r++) v[r] *= by.alpha;
	if (KIND != kNsGram) {
#pragma unroll
		for (int r = 0; r < 16; r++) v[r] += by.beta * ((float)a.hi[r / 4][r % 4] + (float)a.lo[r / 4][r % 4]);
	}
	if (KIND == kNsLast) {
		float* out = reinterpret_cast<float*>(reinterpret_cast<char*>(g.out) + blockIdx.y * g.batch_out);
		const size_t col = col0 + (lane & 31);
#pragma unroll
		for (int r = 0; r < 16; r++) {
			const size_t row = row0 + 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
			if (row < g.out_rows && col < g.out_cols) out[row * g.out_cols + col] = v[r];
		}
	} else {
		char* straight = g.straight + blockIdx.y * g.batch_out + (size_t)row0 * g.straight_stride + (size_t)col0 * 4;
		char* turned = g.turned + blockIdx.y * g.batch_out + (size_t)col0 * g.turned_stride + (size_t)row0 * 4;
		// a tile on the diagonal is its own mirror: each of its elements has one writer
		if ((KIND == kNsGram || KIND == kNsPoly) && diagonal) turned = nullptr;
		store_split_tile(v, corner, straight, g.straight_stride, turned, g.turned_stride);
	}
}

// A group of KS x WP x WQ waves owns a TP x TQ tile of the result. Large products are bound by the matrix pipe and the clock that it
// leaves: X of 4096 x 4096 350 us with tiles of 256 (1180 TFLOP/s of 16-bit products; 320 with everything but the matrix
// instructions left out, 1.8 GHz; the library's product of 16-bit matrices of that size runs at 1330), A 195 and the join 6
// (1060). Below about 2000 the way of a step through group memory and the barrier counts: A of 1003 x 1501 16 us, the pipe busy for 0.28 of
// it. More stages change nothing there (3, 4 and 5: 15.8, 16.2 and 16.0), nor do fragments read one step ahead. KS = 2: two sets of waves, each with one half of every step's
// columns, whose sums meet at the end. With one 32 x 32 tile per wave and as many groups as compute units that puts two
// waves on a SIMD instead of one, and one reads while the other multiplies (A of 1003 x 1501: 18.2 -> 15.9 us).
template <int TP, int TQ, int WP, int WQ, int KS, int STAGES, int KIND>
__global__ __launch_bounds__(WP* WQ* KS * 64) void ns_product_kernel(const NsArgs g) {
	constexpr int kWaves = WP * WQ * KS;
	constexpr int kRows = TP + TQ;
	constexpr int kStage = kRows * kNsBlock;             // bytes of one block of columns of both operands
	constexpr bool kCut = TP <= 128;
	constexpr int kLoads = kRows / (8 * kWaves);         // a load of a wave brings 8 rows
	constexpr int SP = TP / WP / 32, SQ = TQ / WQ / 32;  // 32 x 32 tiles of a wave
	static_assert(kLoads * 8 * kWaves == kRows, "rows divide among the waves");
	static_assert(TP % (8 * kLoads) == 0, "a wave's rows belong to one operand");
	static_assert(STAGES * kStage >= kWaves * 32 * 33 * 4, "the write-out fits the panels' memory, and with KS = 2 the second set's sums (smaller than corners)");
	__shared__ __attribute__((aligned(1024))) char lds[STAGES * kStage];

	const int lane = threadIdx.x & 63;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const NsPair by = pair_of<KIND>(g);
	uint32_t tp, tq;
	uint32_t first = 0, steps = g.k_blocks;
	const bool part = kCut && blockIdx.x >= g.whole;
	if (part) {
		const uint32_t at = blockIdx.x - g.whole, cut = at % g.cuts;
		place_of_tile<KIND>(g, g.whole + at / g.cuts, tp, tq);
		first = cut * g.k_blocks / g.cuts;
		steps = (cut + 1) * g.k_blocks / g.cuts - first;
	} else {
		place_of_tile<KIND>(g, whole_tile_of_group(g), tp, tq);
	}
	const size_t stride = (size_t)g.k_blocks * kNsBlock;
	const char* P = g.P + blockIdx.y * g.batch_p + (size_t)tp * TP * stride + first * kNsBlock;
	const char* Q = g.Q + blockIdx.y * g.batch_q + (size_t)tq * TQ * stride + first * kNsBlock;

	// Row r of a stage lies at 128 r; its 16-byte piece c at place c ^ (r / 2 % 8), so that the 16 lanes that read one
	// piece of 16 rows together meet 16 different quarters of the banks.
	const int first_row = wave * kLoads * 8;
	const char* src = first_row < TP ? P + (size_t)first_row * stride : Q + (size_t)(first_row - TP) * stride;
	uint32_t offset[kLoads];
#pragma unroll
	for (int i = 0; i < kLoads; i++) {
		const uint32_t row = i * 8 + (lane >> 3);
		offset[i] = row * (uint32_t)stride + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
	}
	const uint32_t lds0 = lds_offset(lds) + first_row * kNsBlock;

	// With one 32 x 32 tile per wave every product would wait for the one before: several accumulators in turn.
	constexpr int kChains = SP * SQ == 1 ? 4 / KS : 1;
	floatx16 acc[SP][SQ][kChains];
#pragma unroll
	for (int i = 0; i < SP; i++)
#pragma unroll
		for (int j = 0; j < SQ; j++)
#pragma unroll
			for (int c = 0; c < kChains; c++)
#pragma unroll
				for (int r = 0; r < 16; r++) acc[i][j][c][r] = 0.0f;

	const int ks = wave / (WP * WQ), wp = wave / WQ % WP, wq = wave % WQ;
	const int swizzle = ((lane & 31) >> 1) & 7;
	const char* frag_p = lds + (wp * SP * 32 + (lane & 31)) * kNsBlock;
	const char* frag_q = lds + (TP + wq * SQ * 32 + (lane & 31)) * kNsBlock;

	// A ring of STAGES stages: while one is multiplied, the next STAGES - 1 are on their way.
	uint32_t fetched = 0, fill = 0;  // steps asked for; where the next one goes
	auto fetch = [&]() {
#pragma unroll
		for (int i = 0; i < kLoads; i++) load_to_lds(lds0 + fill + i * 1024, offset[i], src);
		src += kNsBlock;
		fetched++;
		fill = fill + kStage == STAGES * kStage ? 0 : fill + kStage;
	};
	for (int k = 0; k < STAGES - 1; k++)
		if (fetched < steps) fetch();
	uint32_t cur = 0;
	for (uint32_t k = 0; k < steps; k++) {
		// this step's panels are complete when at most the loads of the STAGES - 2 steps behind it are left
		if (fetched - k == STAGES - 1)
			wait_loads<(STAGES - 2) * kLoads>();
		else
			wait_loads<0>();
		__syncthreads();  // everybody's part of the panels is there, and everybody has read the stage before
		if (fetched < steps) fetch();
#pragma unroll
		for (int h0 = 0; h0 < 2 / KS; h0++) {
			const int h = KS == 2 ? ks : h0;
			const int hi_at = ((2 * h + (lane >> 5)) ^ swizzle) << 4, lo_at = hi_at ^ 64;
			half8 p_hi[SP], p_lo[SP], q_hi[SQ], q_lo[SQ];
#pragma unroll
			for (int i = 0; i < SP; i++) {
				p_hi[i] = *reinterpret_cast<const half8*>(frag_p + cur + i * 32 * kNsBlock + hi_at);
				p_lo[i] = *reinterpret_cast<const half8*>(frag_p + cur + i * 32 * kNsBlock + lo_at);
			}
#pragma unroll
			for (int j = 0; j < SQ; j++) {
				q_hi[j] = *reinterpret_cast<const half8*>(frag_q + cur + j * 32 * kNsBlock + hi_at);
				q_lo[j] = *reinterpret_cast<const half8*>(frag_q + cur + j * 32 * kNsBlock + lo_at);
			}
#pragma unroll
			for (int i = 0; i < SP; i++)
#pragma unroll
				for (int j = 0; j < SQ; j++) {
					floatx16& low = acc[i][j][kChains == 4 ? h0 : 0];
					floatx16& high = acc[i][j][kChains == 4 ? 2 + h0 : kChains == 2 ? 1 : 0];
					low = __builtin_amdgcn_mfma_f32_32x32x16_f16(p_lo[i], q_hi[j], low, 0, 0, 0);
					low = __builtin_amdgcn_mfma_f32_32x32x16_f16(p_hi[i], q_lo[j], low, 0, 0, 0);
					high = __builtin_amdgcn_mfma_f32_32x32x16_f16(p_hi[i], q_hi[j], high, 0, 0, 0);
				}
		}
		cur = cur + kStage == STAGES * kStage ? 0 : cur + kStage;
	}
	__syncthreads();  // the panels' memory becomes the waves' corners of the write-out

	uint32_t* corner = reinterpret_cast<uint32_t*>(lds) + wave * 32 * 33;
	const uint32_t p0 = tp * TP + wp * SP * 32, q0 = tq * TQ + wq * SQ * 32;
#pragma unroll
	for (int i = 0; i < SP; i++)
#pragma unroll
		for (int j = 0; j < SQ; j++) {
			const uint32_t row0 = p0 + i * 32, col0 = q0 + j * 32;
			float v[16];
#pragma unroll
			for (int r = 0; r < 16; r++) {
				v[r] = acc[i][j][0][r];
#pragma unroll
				for (int c = 1; c < kChains; c++) v[r] += acc[i][j][c][r];
			}
			if constexpr (KS == 2) {
				static_assert(SP * SQ == 1, "one tile a wave");
				// behind the corners of the write-out: [wave of the first set][4 quarters][lane] of four floats
				float4* other = reinterpret_cast<float4*>(lds + WP * WQ * 32 * 33 * 4) + (wave % (WP * WQ)) * 4 * 64 + lane;
				if (ks == 1)
#pragma unroll
					for (int q = 0; q < 4; q++) other[q * 64] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
				__syncthreads();
				if (ks == 1) return;
#pragma unroll
				for (int q = 0; q < 4; q++) {
					const float4 t = other[q * 64];
					v[4 * q] += t.x;
					v[4 * q + 1] += t.y;
					v[4 * q + 2] += t.z;
					v[4 * q + 3] += t.w;
				}
			}
			if (part) {
				// [tile, part][wave of a set][32 x 32 tile][4 quarters][lane]
				float4* to = g.partial + ((((size_t)(blockIdx.x - g.whole) * WP * WQ + wave) * SP + i) * SQ + j) * 256 + lane;
#pragma unroll
				for (int q = 0; q < 4; q++) to[q * 64] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
				continue;
			}
			Addend a;
			if (KIND != kNsGram) load_addend(g, a, row0, col0);
			finish_tile<KIND>(g, by, v, a, row0, col0, tp == tq, corner);
		}
}

// The tiles that were cut: the parts' sums in their order, and then as a group with the whole tile would go on. A wave per 32 x 32
// tile. T, WP, WQ as in ns_product_kernel.
template <int T, int WP, int WQ, int KIND>
__global__ __launch_bounds__(256) void ns_join_kernel(const NsArgs g) {
	__shared__ uint32_t corner[4][32 * 33];
	constexpr int SP = T / WP / 32, SQ = T / WQ / 32, kTiles = T / 32 * T / 32, kGroups = kTiles / 4;  // 32 x 32 tiles, groups for them
	const int lane = threadIdx.x & 63, corner_of = threadIdx.x >> 6;
	const uint32_t at = blockIdx.x / kGroups, sub = (blockIdx.x % kGroups) * 4 + corner_of;
	const NsPair by = pair_of<KIND>(g);
	uint32_t tp, tq;
	place_of_tile<KIND>(g, g.whole + at, tp, tq);
	const uint32_t wave = sub / (SP * SQ), i = sub / SQ % SP, j = sub % SQ;
	const uint32_t row0 = tp * T + (wave / WQ * SP + i) * 32, col0 = tq * T + (wave % WQ * SQ + j) * 32;
	Addend addend;
	if (KIND != kNsGram) load_addend(g, addend, row0, col0);
	const float4* from = g.partial + ((size_t)at * g.cuts * kTiles + sub) * 256 + lane;
	float v[16];
#pragma unroll
	for (int r = 0; r < 16; r++) v[r] = 0.0f;
#pragma unroll 4
	for (uint32_t c = 0; c < g.cuts; c++, from += kTiles * 256)
#pragma unroll
		for (int q = 0; q < 4; q++) {
			const float4 t = from[q * 64];
			v[4 * q] += t.x;
			v[4 * q + 1] += t.y;
			v[4 * q + 2] += t.z;
			v[4 * q + 3] += t.w;
		}
	finish_tile<KIND>(g, by, v, addend, row0, col0, tp == tq, corner[corner_of]);
}

// Few tiles: what counts is the way from the first load to the last store. A group of eight waves owns a 32 x 32 tile; each
// wave multiplies the whole tile for 16 columns of every step of 128, and the waves' sums meet at the end. A wave fetches
// the rows of one operand for one of a step's four blocks of columns; blocks beyond the end are skipped. (256 x 256, two
// matrices: 5.1 us a product, about half of it the launch's own, against 6.3 with 64 x 64 tiles and one wave per quarter; with one step
// asked for ahead instead of two 5.3, at 512 x 512 7.0 against 6.5. 64 x 64 tiles
// in this form with four | eight waves: A of 1003 x 1501 22 | 16.4 us, X 20.5 | 24.4, where ns_product_kernel takes 15.8 and 19.2.)
// Tiles of 32 are not cut along k between groups: A of a matrix with a short side takes some 0.43 us per 128 of its longer one
// whatever the number of idle units (32 x 2^20 3.5 ms, 64 x 100000 0.3). The chains stay exact enough: 16 x 2^22, one step, 4.8e-7 against
// 64 bits, fp32 products 4.4e-6.
constexpr int kDeepWaves = 8, kDeepStages = 2;
template <int KIND>
__global__ __launch_bounds__(kDeepWaves * 64) void ns_product_deep_kernel(const NsArgs g) {
	constexpr int T = 32, kBlocks = kDeepWaves / 2, kLoads = T / 8;
	constexpr int kPanel = 2 * T * kNsBlock, kStage = kBlocks * kPanel;
	static_assert(kDeepStages * kStage >= kDeepWaves * T * T * 4, "the waves' sums fit the panels' memory, and so does the write-out");
	__shared__ __attribute__((aligned(1024))) char lds[kDeepStages * kStage];
	const int lane = threadIdx.x & 63;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const NsPair by = pair_of<KIND>(g);
	uint32_t tp, tq;
	place_of_tile<KIND>(g, whole_tile_of_group(g), tp, tq);
	const size_t stride = (size_t)g.k_blocks * kNsBlock;
	const uint32_t block = wave >> 1;
	const char* src = (wave & 1 ? g.Q + blockIdx.y * g.batch_q + (size_t)tq * T * stride : g.P + blockIdx.y * g.batch_p + (size_t)tp * T * stride) + block * kNsBlock;
	uint32_t offset[kLoads];
#pragma unroll
	for (int i = 0; i < kLoads; i++) {
		const uint32_t row = i * 8 + (lane >> 3);
		offset[i] = row * (uint32_t)stride + (((lane & 7) ^ ((row >> 1) & 7)) << 4);
	}
	const uint32_t lds0 = lds_offset(lds) + block * kPanel + (wave & 1) * T * kNsBlock;

	const uint32_t steps = (g.k_blocks + kBlocks - 1) / kBlocks;
	auto mine = [&](uint32_t step) { return step * kBlocks + block < g.k_blocks; };  // whether this wave has a part in a step
	uint32_t fill = 0;
	auto fetch = [&](uint32_t step) {
		if (mine(step)) {
#pragma unroll
			for (int i = 0; i < kLoads; i++) load_to_lds(lds0 + fill + i * 1024, offset[i], src);
		}
		src += kBlocks * kNsBlock;
		fill = kStage - fill;
	};
	// Older than the panels' loads, so that the counter that is waited for says nothing of it; it arrives while the products run.
	Addend addend;
	if (KIND != kNsGram && wave == 0) load_addend(g, addend, tp * T, tq * T);
	fetch(0);
	fetch(1);

	floatx16 acc;
#pragma unroll
	for (int r = 0; r < 16; r++) acc[r] = 0.0f;
	const int hi_at = ((2 * (wave & 1) + (lane >> 5)) ^ (((lane & 31) >> 1) & 7)) << 4, lo_at = hi_at ^ 64;
	const char* frag_p = lds + block * kPanel + (lane & 31) * kNsBlock;
	const char* frag_q = frag_p + T * kNsBlock;
	uint32_t cur = 0;
	for (uint32_t k = 0; k < steps; k++) {
		if (mine(k + 1))
			wait_loads<kLoads>();
		else
			wait_loads<0>();
		__syncthreads();  // everybody's part of this step is there
		if (mine(k)) {
			const half8 p_hi = *reinterpret_cast<const half8*>(frag_p + cur + hi_at), p_lo = *reinterpret_cast<const half8*>(frag_p + cur + lo_at);
			const half8 q_hi = *reinterpret_cast<const half8*>(frag_q + cur + hi_at), q_lo = *reinterpret_cast<const half8*>(frag_q + cur + lo_at);
			acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(p_lo, q_hi, acc, 0, 0, 0);
			acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(p_hi, q_lo, acc, 0, 0, 0);
			acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(p_hi, q_hi, acc, 0, 0, 0);
		}
		if (k + 2 < steps) {
			__syncthreads();  // everybody has read this step: its panels' memory takes the step after the next
			fetch(k + 2);
		}
		cur = kStage - cur;
	}
	__syncthreads();

	// the waves' sums: [wave][4 quarters][lane] of four floats
	float4* sums = reinterpret_cast<float4*>(lds);
#pragma unroll
	for (int q = 0; q < 4; q++) sums[(wave * 4 + q) * 64 + lane] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
	__syncthreads();
	if (wave != 0) return;
	float v[16];
#pragma unroll
	for (int q = 0; q < 4; q++) {
		float4 t = sums[q * 64 + lane];
#pragma unroll
		for (int w = 1; w < kDeepWaves; w++) {
			const float4 u = sums[(w * 4 + q) * 64 + lane];
			t.x += u.x;
			t.y += u.y;
			t.z += u.z;
			t.w += u.w;
		}
		v[4 * q] = t.x;
		v[4 * q + 1] = t.y;
		v[4 * q + 2] = t.z;
		v[4 * q + 3] = t.w;
	}
	finish_tile<KIND>(g, by, v, addend, tp * T, tq * T, tp == tq, reinterpret_cast<uint32_t*>(lds));
}

// ---- small matrices: every step in one group ----------------------------------------------------------

// A matrix of at most 64 x 256 (the first and last layers of a small network) stays in the group memory of one compute unit
// from its norm to its last product: X, its transpose and A (then B in its place) in split form, 2 * 64 * NP * 4 B + 16 KiB. One
// launch instead of seventeen, which take 4 to 5 us each however little they compute. us in the kernels, this one | the seventeen:
// one matrix of 64 x 64 17 | 65, 64 x 256 41 | 70, 256 x 3 38 | 67; 64 of 64 x 256 43 | 98, 1000 of them 178 | 490.
// Sixteen waves on 16 x 16 tiles (eight waves on 32 x 32 tiles: 21, 52 and, for the thousand, 268): the products are short, and
// what takes the time between two barriers is the splitting of the results, some fifteen vector instructions an element, and the
// group memory's latency; four waves a SIMD cover each other's.
// The results are written turned (four rows of a lane are four neighbours: 8-byte writes), so X comes from the product
// X^T B and X^T from B X; the second product costs less than the 2-byte writes of the other orientation.
constexpr int kSmallRows = 64, kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr size_t kSmallCols = 256;

struct NsSmallArgs {
	const float* g;
	float* out;
	int m, n;  // rows and columns of X, m <= n
	bool transposed;
	float eps;
	NsSteps steps;
};

// Where piece c (16 bytes: 8 hi or, from c = 4 on, 8 lo) of block kb of a row lies. The sixteen pieces of two blocks are
// exchanged by the row, so that the lanes that read one piece of 16 rows meet different banks.
__device__ __forceinline__ int small_at(int row, int row_bytes, int kb, int c) { return row * row_bytes + (kb >> 1) * 256 + ((((kb & 1) * 8 + c) ^ (row & 15)) << 4); }

template <int NP>
__global__ __launch_bounds__(kSmallThreads) void ns_small_kernel(const NsSmallArgs a) {
	constexpr int kX = 0, kXt = kSmallRows * NP * 4, kA = 2 * kXt;  // byte offsets
	constexpr int kRowX = NP * 4, kRowM = kSmallRows * 4;           // bytes of a row of X; of X^T and A
	__shared__ __attribute__((aligned(256))) char lds[kA + kSmallRows * kSmallRows * 4];
	__shared__ double red[kSmallWaves];
	__shared__ NsFactors own_factors[64];  // of a matrix far below eps
	const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quarter = lane >> 4;
	const int m = a.m, n = a.n;
	const float* g = a.g + (size_t)blockIdx.x * m * n;

	// two rows by two columns of X per thread and turn
	constexpr int kTurns = kSmallRows * NP / 4 / kSmallThreads;
	float v[kTurns][4];
	double sum = 0.0;
#pragma unroll
	for (int t = 0; t < kTurns; t++) {
		const int at = t * kSmallThreads + tid, r0 = at / (NP / 2) * 2, c0 = at % (NP / 2) * 2;
#pragma unroll
		for (int k = 0; k < 4; k++) {
			const int r = r0 + (k >> 1), c = c0 + (k & 1);
			v[t][k] = r < m && c < n ? (a.transposed ? g[(size_t)c * m + r] : g[(size_t)r * n + c]) : 0.0f;
			sum += (double)v[t][k] * (double)v[t][k];
		}
	}
	sum = wave_reduce(sum, [](double x, double y) { return x + y; });
	if (lane == 0) red[wave] = sum;
	__syncthreads();
	sum = 0.0;
#pragma unroll
	for (int w = 0; w < kSmallWaves; w++) sum += red[w];
	const double own = sqrt(sum), norm = own + (double)a.eps, first = ns_first_bound(own, a.eps);
	const double factor = !isfinite(norm) ? (double)nanf("") : norm > 0.0 ? scale_for(first) / norm : 0.0;
	const bool usual = __builtin_amdgcn_readfirstlane(first == 1.0);
	if (!usual && tid == 0) ns_own_factors(a.steps, first, own_factors);
#pragma unroll
	for (int t = 0; t < kTurns; t++) {
		const int at = t * kSmallThreads + tid, r0 = at / (NP / 2) * 2, c0 = at % (NP / 2) * 2;
		uint32_t p[4];
#pragma unroll
		for (int k = 0; k < 4; k++) p[k] = split_pair((float)((double)v[t][k] * factor));
#pragma unroll
		for (int k = 0; k < 2; k++) {
			// row r0 + k of X, columns c0 and c0 + 1; row c0 + k of X^T, columns r0 and r0 + 1
			const uint32_t x0 = p[2 * k], x1 = p[2 * k + 1], t0 = p[k], t1 = p[2 + k];
			char* to = lds + kX + (c0 & 7) * 2;
			*reinterpret_cast<uint32_t*>(to + small_at(r0 + k, kRowX, c0 >> 5, (c0 & 31) >> 3)) = (x0 & 0xFFFFu) | (x1 << 16);
			*reinterpret_cast<uint32_t*>(to + small_at(r0 + k, kRowX, c0 >> 5, ((c0 & 31) >> 3) + 4)) = (x0 >> 16) | (x1 & 0xFFFF0000u);
			to = lds + kXt + (r0 & 7) * 2;
			*reinterpret_cast<uint32_t*>(to + small_at(c0 + k, kRowM, r0 >> 5, (r0 & 31) >> 3)) = (t0 & 0xFFFFu) | (t1 << 16);
			*reinterpret_cast<uint32_t*>(to + small_at(c0 + k, kRowM, r0 >> 5, ((r0 & 31) >> 3) + 4)) = (t0 >> 16) | (t1 & 0xFFFF0000u);
		}
	}
	__syncthreads();

	// A lane's row of a tile is lane % 16 (tiles begin at multiples of 16), so what small_at exchanges by is the lane's own: the
	// address of a piece is a lane's part, one exclusive or with a constant, and an offset that the wave shares. Operands:
	// 8 columns per quarter of a wave (piece `quarter`). Results: element i of a lane is row 4 quarter + i, column lane % 16.
	int lane_x = (lane & 15) * kRowX, lane_m = (lane & 15) * kRowM, row_turn = (lane & 15) << 4, read_at = row_turn ^ (quarter << 4);
	struct Operand {
		half8 hi, lo;
	};
	auto read = [&](int P, int p_bytes, int p0, int kb) {
		const char* p = lds + P + p0 * p_bytes + (p_bytes == kRowX ? lane_x : lane_m) + (kb >> 1) * 256;
		const int turn = read_at ^ ((kb & 1) << 7);
		Operand o;
		o.hi = *reinterpret_cast<const half8*>(p + turn);
		o.lo = *reinterpret_cast<const half8*>(p + (turn ^ 64));
		return o;
	};
	// X and X^T are two copies that are carried on separately: the same element of both has to come out with the same bits. A difference
	// between them, d, becomes a d in every step, however far X has converged (64 x 64, the quintic: no digit was left after 20
	// steps). So an element is the same terms in the same order in both, whichever operand holds them: `turned` exchanges the two products
	// with low halves along with the operands, and what is added afterwards leaves the compiler no choice of its roundings.
	auto multiply = [&](floatx4& low, floatx4& high, const Operand& p, const Operand& q, auto turned) {
		low = __builtin_amdgcn_mfma_f32_16x16x32_f16(turned ? p.hi : p.lo, turned ? q.lo : q.hi, low, 0, 0, 0);
		high = __builtin_amdgcn_mfma_f32_16x16x32_f16(p.hi, q.hi, high, 0, 0, 0);
		low = __builtin_amdgcn_mfma_f32_16x16x32_f16(turned ? p.lo : p.hi, turned ? q.hi : q.lo, low, 0, 0, 0);
	};
	// where a lane's four rows of the tile (p0, q0) lie in D, which holds the result turned: D[q0 + lane's column][p0 + rows]
	auto place = [&](int D, int d_bytes, int p0, int q0) {
		const int s = ((p0 >> 5) & 1) * 8 + ((p0 & 16) >> 3) + (quarter >> 1);
		return lds + D + q0 * d_bytes + (d_bytes == kRowX ? lane_x : lane_m) + (p0 >> 6) * 256 + (row_turn ^ (s << 4)) + (quarter & 1) * 8;
	};
	// r = alpha r + beta D
	auto add = [&](floatx4& r, float alpha, float beta, int D, int d_bytes, int p0, int q0) {
		const char* d = place(D, d_bytes, p0, q0);
		const half4 hi = *reinterpret_cast<const half4*>(d), lo = *reinterpret_cast<const half4*>(reinterpret_cast<const char*>(lds) + ((d - lds) ^ 64));
#pragma unroll
		for (int i = 0; i < 4; i++) r[i] = __builtin_fmaf(alpha, r[i], beta * ((float)hi[i] + (float)lo[i]));
	};
	auto store = [&](const floatx4& r, int D, int d_bytes, int p0, int q0) {
		char* d = place(D, d_bytes, p0, q0);
		uint32_t s[4];
#pragma unroll
		for (int i = 0; i < 4; i++) s[i] = split_pair(r[i]);
		*reinterpret_cast<uint2*>(d) = make_uint2((s[0] & 0xFFFFu) | (s[1] << 16), (s[2] & 0xFFFFu) | (s[3] << 16));
		*reinterpret_cast<uint2*>(lds + ((d - lds) ^ 64)) = make_uint2((s[0] >> 16) | (s[1] & 0xFFFF0000u), (s[2] >> 16) | (s[3] & 0xFFFF0000u));
	};

	// addresses are worked out anew where they are used: all of them, kept, would take more than the 128 registers of a lane
	auto forget = [&] { asm volatile("" : "+v"(lane_x), "+v"(lane_m), "+v"(row_turn), "+v"(read_at) :: "memory"); };

	const int ti = (wave >> 2) * 16, tj = (wave & 3) * 16;  // this wave's tile of A and B
	constexpr int kShare = NP / 32;                         // and its tiles of X and of X^T: 2 * 4 * NP / 16 among sixteen
	auto uniform = [](float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v))); };
	for (int k = 0; k < a.steps.count; k++) {
		NsFactors by;
		if (usual)
			by = a.steps.usual[k];
		else
			by = {uniform(own_factors[k].gram), uniform(own_factors[k].poly), uniform(own_factors[k].poly_a), uniform(own_factors[k].update), uniform(own_factors[k].update_x)};
		forget();
		floatx4 low = {0.0f, 0.0f, 0.0f, 0.0f}, high = low;
#pragma unroll 4
		for (int kb = 0; kb < NP / 32; kb++) multiply(low, high, read(kX, kRowX, ti, kb), read(kX, kRowX, tj, kb), std::false_type());
		floatx4 r = by.gram * (low + high);
		store(r, kA, kRowM, ti, tj);
		__syncthreads();
		// B in A's place
		low = high = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
		for (int kb = 0; kb < 2; kb++) multiply(low, high, read(kA, kRowM, ti, kb), read(kA, kRowM, tj, kb), std::false_type());
		r = low + high;
		add(r, by.poly, by.poly_a, kA, kRowM, ti, tj);
		__syncthreads();
		store(r, kA, kRowM, ti, tj);
		__syncthreads();
		// X: waves 0 .. 7 the tiles of B X (written to X^T), the others those of X^T B (written to X); a wave has one of the four
		// rows of tiles of B and every second one of X^T
		const bool last = k + 1 == a.steps.count;
		const int form = wave >> 3, mi = (wave & 3) * 16, n0 = (wave >> 2) & 1;
		floatx4 x[kShare];
		auto multiply_x = [&](auto which) {
			constexpr bool kTurned = which;
			const Operand b0 = read(kA, kRowM, mi, 0), b1 = read(kA, kRowM, mi, 1);
#pragma unroll
			for (int i = 0; i < kShare; i++) {
				const int ni = (2 * i + n0) * 16;
				low = high = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
				const Operand x0 = read(kXt, kRowM, ni, 0), x1 = read(kXt, kRowM, ni, 1);
				multiply(low, high, kTurned ? x0 : b0, kTurned ? b0 : x0, which);
				multiply(low, high, kTurned ? x1 : b1, kTurned ? b1 : x1, which);
				x[i] = low + high;
				if constexpr (kTurned)
					add(x[i], by.update, by.update_x, kX, kRowX, ni, mi);
				else
					add(x[i], by.update, by.update_x, kXt, kRowM, mi, ni);
				forget();
			}
		};
		auto store_x = [&](auto which) {
#pragma unroll
			for (int i = 0; i < kShare; i++) {
				const int ni = (2 * i + n0) * 16;
				if constexpr (which)
					store(x[i], kX, kRowX, ni, mi);
				else
					store(x[i], kXt, kRowM, mi, ni);
				forget();
			}
		};
		if (!last) {
			form ? multiply_x(std::true_type()) : multiply_x(std::false_type());
			__syncthreads();
			form ? store_x(std::true_type()) : store_x(std::false_type());
			__syncthreads();
		} else if (form == (int)a.transposed) {
			form ? multiply_x(std::true_type()) : multiply_x(std::false_type());
			// out has the rows and columns of g: those of X, or of X^T
			const int rows = a.transposed ? n : m, cols = a.transposed ? m : n;
			float* out = a.out + (size_t)blockIdx.x * m * n;
			int row = 4 * quarter, col = lane & 15;
			asm volatile("" : "+v"(row), "+v"(col));
#pragma unroll
			for (int i = 0; i < kShare; i++) {
				const int ni = (2 * i + n0) * 16, row0 = (a.transposed ? ni : mi) + row, col0 = (a.transposed ? mi : ni) + col;
#pragma unroll
				for (int j = 0; j < 4; j++)
					if (row0 + j < rows && col0 < cols) out[(row0 + j) * cols + col0] = x[i][j];
			}
		}
	}
}

// ---- the host's side --------------------------------------------------------------------------------

// The tile of a product whose result is m x n (half of m x m for the symmetric kinds). A larger tile reads less per product
// but leaves compute units idle. The measured time of a step of 32 columns over all of the result is close to a line in the
// number n of tiles, in ns on 256 units: 130 + 0.5 n with tiles of 32, 220 + 1.1 n with 64, 500 + 2.7 n with 128, and
// 3.3 n + 1900 for each round of the units with 256, of which only one fits a unit. The smallest wins. Measured, us per
// product, smaller | larger tile:
//   32 | 64:   X of 768 x 768 14.7 | 12.0, its A 9.2 | 11.7;      64 | 128: A of 2048 x 2048 45 | 54, its X 76.5 | 64.7
//   128 | 256: X of 3000 x 3000 206 | 212, of 4096 x 4096 388 | 354; its A 251 | 262 (136 tiles of 256 on 256 units)
static int ns_tile(size_t m, size_t n, bool half, size_t batch) {
	static const int tiles[4] = {32, 64, 128, 256};
	static const double base[4] = {130.0, 220.0, 500.0, 1900.0}, slope[4] = {0.5, 1.1, 2.7, 3.3};
	int best = 0;
	double least = 0.0;
	for (int i = 0; i < 4; i++) {
		const size_t tm = (m + tiles[i] - 1) / tiles[i], tn = (n + tiles[i] - 1) / tiles[i];
		const double count = (double)batch * (half ? tm * (tm + 1) / 2 : tm * tn) * 256.0 / state().compute_units;
		const double time = base[i] * (i == 3 ? ceil(count / 256.0) : 1.0) + slope[i] * count;
		if (i == 0 || time < least) {
			least = time;
			best = tiles[i];
		}
	}
	return best;
}

// Tiles that are left over when every compute unit has had the same number keep few units busy for the time of a whole tile:
// into how many parts along k each of them is cut (1: not), `left` receiving their number. By the measured time of a step of
// the tiles that a unit works on, the parts' way through memory at 5 TB/s and 6 us for the join; it has to save a seventh of
// the round. us per product, cut, with the join | whole: A of 4096 x 4096 (528 tiles of 128) 202 | 239, of 3000 x 3000 (300)
// 96 | 115, X of 3000 x 3000 (576) 171 | 201; not cut: A of 3500 x 3500 (406) 148 | 144. Three tiles of 64 share a unit and the
// first two hardly slow each other, so those are cut from two rounds on: A of 2000 x 4100 (528 tiles of 64) 76 | 88, of 2048 x 2048
// 42.5 | 44; not cut: A of 1500 x 3000 (300) 44 | 41.
static unsigned ns_cuts(size_t tiles, int tile, uint32_t k_blocks, size_t batch, size_t& left) {
	const size_t units = state().compute_units;
	left = tiles % units;
	if (batch != 1 || left == 0 || !(tile == 128 || (tile == 64 && tiles >= 2 * units))) return 1;
	const double round = (tile == 128 ? 0.69 : 0.28) * k_blocks, part = tile * tile * 1.6e-6;  // us
	double least = 0.85 * round;
	unsigned best = 1;
	for (unsigned c = 2; c <= 16 && k_blocks / c >= 4; c++) {
		const double time = round * ((left * c + units - 1) / units) / c + left * c * part + 6.0;
		if (time < least) {
			least = time;
			best = c;
		}
	}
	return best;
}

static size_t ns_tiles(size_t p_rows, size_t q_rows, int tile, bool half) {
	const size_t tp = p_rows / tile, tq = q_rows / tile;
	return half ? tp * (tp + 1) / 2 : tp * tq;
}

// Bytes that the parts of a product's cut tiles take.
static size_t ns_partial_bytes(size_t p_rows, size_t q_rows, int tile, bool half, uint32_t k_blocks, size_t batch) {
	size_t left;
	const unsigned cuts = ns_cuts(ns_tiles(p_rows, q_rows, tile, half), tile, k_blocks, batch, left);
	return cuts > 1 ? left * cuts * tile * tile * sizeof(float) : 0;
}

template <int KIND>
static int ns_product(const NsArgs& args, int tile, size_t p_rows, size_t q_rows, size_t batch) {
	constexpr bool kHalf = KIND == kNsGram || KIND == kNsPoly;
	NsArgs a = args;
	a.tiles_p = (uint32_t)(p_rows / tile);
	a.tiles_q = (uint32_t)(q_rows / tile);
	const unsigned tiles = (unsigned)ns_tiles(p_rows, q_rows, tile, kHalf);
	size_t left = 0;
	a.cuts = ns_cuts(tiles, tile, a.k_blocks, batch, left);
	if (a.cuts == 1) left = 0;
	a.whole = tiles - (unsigned)left;
	a.band = (uint32_t)sqrt(tiles / 8.0);
	if (a.band < 1) a.band = 1;
	const dim3 grid(a.whole + (unsigned)left * a.cuts, (unsigned)batch);
	hipStream_t stream = state().stream;
	switch (tile) {
		case 32: hipLaunchKernelGGL(ns_product_deep_kernel<KIND>, grid, dim3(kDeepWaves * 64), 0, stream, a); break;
		case 64: hipLaunchKernelGGL((ns_product_kernel<64, 64, 2, 2, 2, 3, KIND>), grid, dim3(512), 0, stream, a); break;
		case 128: hipLaunchKernelGGL((ns_product_kernel<128, 128, 2, 4, 1, 2, KIND>), grid, dim3(512), 0, stream, a); break;
		default: hipLaunchKernelGGL((ns_product_kernel<256, 256, 2, 4, 1, 2, KIND>), grid, dim3(512), 0, stream, a); break;
	}
	TFHIP_CHECK_LAUNCH();
	if (left) {
		if (tile == 64)
			hipLaunchKernelGGL((ns_join_kernel<64, 2, 2, KIND>), dim3((unsigned)left), dim3(256), 0, stream, a);
		else
			hipLaunchKernelGGL((ns_join_kernel<128, 2, 4, KIND>), dim3((unsigned)left * 4), dim3(256), 0, stream, a);
		TFHIP_CHECK_LAUNCH();
	}
	return TFHIP_OK;
}

static NsSteps ns_steps(int count, const float* coefficients) {
	NsSteps s = {};
	s.count = count;
	NsScales scales(1.0);
	for (int k = 0; k < count; k++) {
		for (int i = 0; i < 3; i++) s.coefficients[k][i] = coefficients[3 * k + i];
		s.usual[k] = scales.step(s.coefficients[k], k + 1 == count);
	}
	return s;
}

static int newton_schulz_small(const float* g, float* out, size_t batch, size_t rows, size_t cols, const NsSteps& steps, float eps) {
	NsSmallArgs args = {};
	args.g = g;
	args.out = out;
	args.transposed = rows > cols;
	args.m = (int)(args.transposed ? cols : rows);
	args.n = (int)(args.transposed ? rows : cols);
	args.eps = eps;
	args.steps = steps;
	const dim3 grid((unsigned)batch), block(kSmallThreads);
	if (args.n <= 64)
		hipLaunchKernelGGL(ns_small_kernel<64>, grid, block, 0, state().stream, args);
	else if (args.n <= 128)
		hipLaunchKernelGGL(ns_small_kernel<128>, grid, block, 0, state().stream, args);
	else
		hipLaunchKernelGGL(ns_small_kernel<256>, grid, block, 0, state().stream, args);
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}

static bool ns_fits_one_group(size_t shorter, size_t longer) { return shorter <= (size_t)kSmallRows && longer <= kSmallCols; }

struct NsPlan {
	int tile_half, tile_full;  // of the symmetric products and of the others
	size_t mp, np;             // padded sides
	size_t at_once;            // matrices, as many as a work space of 4 GiB holds, at least one
};
static NsPlan ns_plan(size_t batch, size_t m, size_t n) {
	NsPlan p;
	const size_t counted = batch < 256 ? batch : 256;
	p.tile_half = ns_tile(m, m, true, counted);
	p.tile_full = ns_tile(m, n, false, counted);
	const size_t tile = p.tile_half > p.tile_full ? p.tile_half : p.tile_full;
	p.mp = (m + tile - 1) / tile * tile;
	p.np = (n + tile - 1) / tile * tile;
	p.at_once = std::max<size_t>(1, ((size_t)4 << 30) / (16 * p.mp * p.np + 8 * p.mp * p.mp));
	return p;
}

// `batch` matrices whose work space fits the arena together.
static int newton_schulz(const float* g, float* out, size_t batch, size_t rows, size_t cols, const NsSteps& steps, float eps, const NsPlan& plan) {
	State& s = state();
	const int tile_half = plan.tile_half, tile_full = plan.tile_full;
	const size_t mp = plan.mp, np = plan.np;
	const bool transposed = rows > cols;
	const size_t m = transposed ? cols : rows, n = transposed ? rows : cols, elements = rows * cols;
	// a group takes four vectors a thread, or, where there are none, four elements (30 of 101 x 75: 9.6 -> 3.5 us, 1501 x 1003 6.6 -> 5.0)
	const bool vec = (elements & 3) == 0 && ((uintptr_t)g & 15) == 0;
	const size_t share = vec ? 4096 : 1024, shares = elements / share;
	const unsigned parts = (unsigned)(shares < 1 ? 1 : shares < 512 ? shares : 512);
	auto align = [](size_t b) { return (b + 255) & ~size_t(255); };
	const size_t norm_bytes = align(batch * parts * sizeof(double)), factor_bytes = align(batch * steps.count * sizeof(NsFactors)), x_bytes = align(batch * mp * np * 4), a_bytes = align(batch * mp * mp * 4);
	const uint32_t blocks_m = (uint32_t)(mp / kNsStep), blocks_n = (uint32_t)(np / kNsStep);
	const size_t parts_bytes[3] = {ns_partial_bytes(mp, mp, tile_half, true, blocks_n, batch), ns_partial_bytes(mp, mp, tile_half, true, blocks_m, batch),
	                               ns_partial_bytes(mp, np, tile_full, false, blocks_m, batch)};
	const size_t partial_bytes = std::max({parts_bytes[0], parts_bytes[1], parts_bytes[2]});
	char* base = (char*)scratch(norm_bytes + factor_bytes + 4 * x_bytes + 2 * a_bytes + partial_bytes);
	if (!base) return TFHIP_ERR_HIP;
	double* partial = (double*)base;
	NsFactors* factors = (NsFactors*)(base + norm_bytes);
	char* x = base + norm_bytes + factor_bytes;
	char* xt = x + x_bytes;
	char* x_next = xt + x_bytes;
	char* xt_next = x_next + x_bytes;
	char* A = xt_next + x_bytes;
	char* B = A + a_bytes;
	float4* products_partial = (float4*)(B + a_bytes);

	hipLaunchKernelGGL(ns_norm_kernel, dim3((unsigned)batch * parts), dim3(256), 0, s.stream, g, partial, elements, parts, vec);
	TFHIP_CHECK_LAUNCH();
	const size_t split_groups = (mp / 32 * (np / 32) + 3) / 4, most = (size_t)s.compute_units * 8;
	hipLaunchKernelGGL(ns_split_kernel, dim3((unsigned)(split_groups < most ? split_groups : most), (unsigned)batch), dim3(256), 0, s.stream, g, (const double*)partial, parts, x, xt, m, n, mp, np, transposed, eps,
	                   factors, steps);
	TFHIP_CHECK_LAUNCH();
	for (int k = 0; k < steps.count; k++) {
		NsArgs gram = {};
		gram.factors = factors + k;
		gram.steps = (uint32_t)steps.count;
		gram.P = gram.Q = x;
		gram.straight = gram.turned = A;
		gram.straight_stride = gram.turned_stride = mp * 4;
		gram.batch_p = gram.batch_q = mp * np * 4;
		gram.batch_out = mp * mp * 4;
		gram.partial = products_partial;
		gram.k_blocks = blocks_n;
		int rc = ns_product<kNsGram>(gram, tile_half, mp, mp, batch);
		if (rc) return rc;
		NsArgs poly = gram;
		poly.P = poly.Q = poly.addend = A;
		poly.straight = poly.turned = B;
		poly.batch_p = poly.batch_q = poly.batch_addend = mp * mp * 4;
		poly.addend_stride = mp * 4;
		poly.k_blocks = blocks_m;
		rc = ns_product<kNsPoly>(poly, tile_half, mp, mp, batch);
		if (rc) return rc;
		const bool last = k + 1 == steps.count;
		const bool turn = last && transposed;  // the caller's rows are the columns of X
		NsArgs update = {};
		update.P = turn ? xt : B;
		update.Q = turn ? B : xt;
		update.batch_p = turn ? mp * np * 4 : mp * mp * 4;
		update.batch_q = turn ? mp * mp * 4 : mp * np * 4;
		update.addend = turn ? x : xt;
		update.addend_stride = (turn ? np : mp) * 4;
		update.batch_addend = mp * np * 4;
		update.partial = products_partial;
		update.factors = gram.factors;
		update.steps = gram.steps;
		update.k_blocks = blocks_m;
		if (last) {
			update.out = out;
			update.out_rows = rows;
			update.out_cols = cols;
			update.batch_out = elements * sizeof(float);
			rc = ns_product<kNsLast>(update, tile_full, turn ? np : mp, turn ? mp : np, batch);
		} else {
			update.straight = x_next;
			update.turned = xt_next;
			update.straight_stride = np * 4;
			update.turned_stride = mp * 4;
			update.batch_out = mp * np * 4;
			rc = ns_product<kNsUpdate>(update, tile_full, mp, np, batch);
		}
		if (rc) return rc;
		char* t = x;
		x = x_next;
		x_next = t;
		t = xt;
		xt = xt_next;
		xt_next = t;
	}
	return TFHIP_OK;
}

}  // namespace tfhip

using namespace tfhip;

extern "C" int tfhip_newton_schulz_f32(const float* g, float* out, size_t batch, size_t rows, size_t cols, int steps, const float* coefficients, float eps) {
	if (rows == 0 || cols == 0) return fail(TFHIP_ERR_ARG, "orthogonalisation of an empty matrix (%zu x %zu)", rows, cols);
	const size_t shorter = rows < cols ? rows : cols, longer = rows < cols ? cols : rows;
	if (shorter > 32768 || longer > 0x7FFFFF || rows * cols > 0x7FFFFFFF)
		return fail(TFHIP_ERR_ARG, "orthogonalisation of a %zu x %zu matrix: at most 32768 on its shorter side, 2^23 - 1 on its longer one and 2^31 - 1 elements", rows, cols);
	if (batch > 65535) return fail(TFHIP_ERR_ARG, "more than 65535 matrices in one batch (%zu)", batch);
	if (steps < 1 || steps > 64) return fail(TFHIP_ERR_ARG, "%d Newton-Schulz steps (1 to 64 are taken)", steps);
	if (!coefficients) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_newton_schulz_f32");
	for (int i = 0; i < 3 * steps; i++)
		if (!isfinite(coefficients[i])) return fail(TFHIP_ERR_ARG, "coefficient %d of the Newton-Schulz steps is not finite", i);
	if (!(eps >= 0.0f) || !isfinite(eps)) return fail(TFHIP_ERR_ARG, "Newton-Schulz with eps = %g: a finite number of at least 0 is needed", (double)eps);
	if (batch == 0) return TFHIP_OK;
	if (!g || !out) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_newton_schulz_f32");
	if (g != out && words_overlap(g, batch * rows * cols, out, batch * rows * cols)) return fail(TFHIP_ERR_ARG, "Newton-Schulz: g and out overlap without being the same");
	TFHIP_REQUIRE_INIT();
	TFHIP_HOLD_DEVICE();
	const NsSteps taken = ns_steps(steps, coefficients);
	if (ns_fits_one_group(shorter, longer)) return newton_schulz_small(g, out, batch, rows, cols, taken, eps);
	const NsPlan plan = ns_plan(batch, shorter, longer);
	for (size_t first = 0; first < batch; first += plan.at_once) {
		const size_t count = batch - first < plan.at_once ? batch - first : plan.at_once;
		const int rc = newton_schulz(g + first * rows * cols, out + first * rows * cols, count, rows, cols, taken, eps, plan);
		if (rc) return rc;
	}
	return TFHIP_OK;
}

extern "C" int tfhip_test_newton_schulz_tiles(size_t batch, size_t rows, size_t cols, int* tiles, unsigned* cuts) {
	TFHIP_REQUIRE_INIT();
	const size_t shorter = rows < cols ? rows : cols, longer = rows < cols ? cols : rows;
	if (!tiles || !cuts || batch == 0 || shorter == 0) return fail(TFHIP_ERR_ARG, "null pointer or empty batch passed to tfhip_test_newton_schulz_tiles");
	tiles[0] = tiles[1] = 0;
	cuts[0] = cuts[1] = cuts[2] = 1;
	if (ns_fits_one_group(shorter, longer)) return TFHIP_OK;
	const NsPlan plan = ns_plan(batch, shorter, longer);
	const size_t count = batch < plan.at_once ? batch : plan.at_once;
	const uint32_t blocks_m = (uint32_t)(plan.mp / kNsStep), blocks_n = (uint32_t)(plan.np / kNsStep);
	size_t left;
	tiles[0] = plan.tile_half;
	tiles[1] = plan.tile_full;
	cuts[0] = ns_cuts(ns_tiles(plan.mp, plan.mp, plan.tile_half, true), plan.tile_half, blocks_n, count, left);
	cuts[1] = ns_cuts(ns_tiles(plan.mp, plan.mp, plan.tile_half, true), plan.tile_half, blocks_m, count, left);
	cuts[2] = ns_cuts(ns_tiles(plan.mp, plan.np, plan.tile_full, false), plan.tile_full, blocks_m, count, left);
	return TFHIP_OK;
}
