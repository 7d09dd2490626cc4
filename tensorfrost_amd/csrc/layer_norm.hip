// Layer norm of the rows of a matrix, and its backward pass.
//
//   mu = mean_c x,  s = 1 / sqrt(mean_c (x - mu)^2 + eps),  xhat = (x - mu) s,  y = xhat w + b
//   g = dy w,  dx = s (g - mean_c g - xhat mean_c(g xhat)),  dw = sum_r dy xhat,  db = sum_r dy
//
// The reference has no such operation; a user composes it from the mean and norm reductions
// (TensorFrost/Compiler/Implementations.cpp:243-303) and element-wise kernels, as for the softmax.
// The variance is taken about the mean that was just computed (two sums, not the difference of two large ones), so a row
// whose mean is large against its spread keeps its digits. All sums are fp32.

#include "common.h"

#include <math.h>

#include <type_traits>

namespace tfhip {

constexpr int kLnThreads = 256;

// How a row is moved. Whole: four floats at once, rows of whole vectors on 16-byte addresses. Otherwise either Single floats,
// or Anywhere: vectors on 4-byte addresses, which the memory pipeline takes too, the last one of a row element by element.
// A vector that crosses a cache line costs two; long rows, with 16 floats a thread of a large block, gain more from fewer
// instructions, short ones do not. Single | Anywhere, us: forward 4096 x 16383 146 | 109, 8192 x 5001 80 | 68, 65536 x 250 28 | 30,
// 4099 x 1001 7.6 | 8.0; backward 4096 x 16383 187 | 160, 8192 x 5001 116 | 122, 65536 x 250 37 | 44.
enum class Access { Whole, Anywhere, Single };
typedef float LnVec __attribute__((ext_vector_type(4)));
typedef float LnVecAnywhere __attribute__((ext_vector_type(4), aligned(4)));
template <Access ACCESS>
using LnVecAt = std::conditional_t<ACCESS == Access::Whole, LnVec, LnVecAnywhere>;

// Which element of the row is element i of a thread: vectors, or single floats, GROUP of them apart.
template <int GROUP, Access ACCESS>
__device__ __forceinline__ int place(int i, int lane) {
	return ACCESS == Access::Single ? i * GROUP + lane : (i / 4 * GROUP + lane) * 4 + i % 4;
}
template <int GROUP, Access ACCESS>
__device__ __forceinline__ bool inside(int i, int lane, int cols) {
	return place<GROUP, ACCESS>(ACCESS == Access::Whole ? i / 4 * 4 : i, lane) < cols;
}

// E elements of a row per thread of a GROUP; `empty` beyond the row. KEPT: what every row uses and the caches should hold; `p`
// may then be null.
template <int GROUP, int E, Access ACCESS, bool KEPT>
__device__ __forceinline__ void load_elements(const float* p, float (&v)[E], int lane, int cols, float empty) {
	typedef LnVecAt<ACCESS> Vec;
	if constexpr (ACCESS == Access::Single) {
#pragma unroll
		for (int i = 0; i < E; i++) {
			const int c = place<GROUP, ACCESS>(i, lane);
			v[i] = (!KEPT || p) && c < cols ? KEPT ? p[c] : __builtin_nontemporal_load(p + c) : empty;
		}
	} else {
#pragma unroll
		for (int i = 0; i < E; i += 4) {
			const int c = place<GROUP, ACCESS>(i, lane);
			LnVec t = LnVec(empty);
			if (!KEPT || p) {
				if (ACCESS == Access::Whole ? c < cols : c + 4 <= cols) {
					t = KEPT ? *reinterpret_cast<const Vec*>(p + c) : __builtin_nontemporal_load(reinterpret_cast<const Vec*>(p + c));
				} else if (ACCESS == Access::Anywhere && c < cols) {
#pragma unroll
					for (int j = 0; j < 3; j++)
						if (c + j < cols) t[j] = p[c + j];
				}
			}
#pragma unroll
			for (int j = 0; j < 4; j++) v[i + j] = t[j];
		}
	}
}
template <int GROUP, int E, Access ACCESS>
__device__ __forceinline__ void load_row(const float* p, float (&v)[E], int lane, int cols) {
	load_elements<GROUP, E, ACCESS, false>(p, v, lane, cols, 0.0f);
}
template <int GROUP, int E, Access ACCESS>
__device__ __forceinline__ void load_shared(const float* p, float (&v)[E], int lane, int cols, float empty) {
	load_elements<GROUP, E, ACCESS, true>(p, v, lane, cols, empty);
}
// STREAM: past the caches.
template <int GROUP, int E, Access ACCESS, bool STREAM>
__device__ __forceinline__ void store_row(float* p, const float (&v)[E], int lane, int cols) {
	typedef LnVecAt<ACCESS> Vec;
	if constexpr (ACCESS == Access::Single) {
#pragma unroll
		for (int i = 0; i < E; i++) {
			const int c = place<GROUP, ACCESS>(i, lane);
			if (c >= cols) continue;
			if (STREAM)
				__builtin_nontemporal_store(v[i], p + c);
			else
				p[c] = v[i];
		}
	} else {
#pragma unroll
		for (int i = 0; i < E; i += 4) {
			const int c = place<GROUP, ACCESS>(i, lane);
			LnVec t;
#pragma unroll
			for (int j = 0; j < 4; j++) t[j] = v[i + j];
			if (ACCESS == Access::Whole ? c < cols : c + 4 <= cols) {
				if (STREAM)
					__builtin_nontemporal_store(t, reinterpret_cast<Vec*>(p + c));
				else
					*reinterpret_cast<Vec*>(p + c) = t;
			} else if (ACCESS == Access::Anywhere && c < cols) {
#pragma unroll
				for (int j = 0; j < 3; j++)
					if (c + j < cols) p[c + j] = t[j];
			}
		}
	}
}

// N sums over the threads of a GROUP at once, in every thread. Up to a wave by exchanges; larger groups (the whole
// block) through group memory, `red` with room for N * GROUP / 64 floats that no other call in flight uses.
template <int GROUP, int N>
__device__ __forceinline__ void group_sums(float (&v)[N], float* red) {
#pragma unroll
	for (int off = (GROUP < 64 ? GROUP : 64) / 2; off >= 1; off >>= 1)
#pragma unroll
		for (int i = 0; i < N; i++) v[i] += __shfl_xor(v[i], off, 64);
	if constexpr (GROUP > 64) {
		if ((threadIdx.x & 63) == 0)
#pragma unroll
			for (int i = 0; i < N; i++) red[(threadIdx.x >> 6) * N + i] = v[i];
		__syncthreads();
		if constexpr (GROUP >= 512 && N == 1) {  // by exchanges again, which keeps the registers
			float t = red[threadIdx.x & (GROUP / 64 - 1)];
#pragma unroll
			for (int off = GROUP / 128; off >= 1; off >>= 1) t += __shfl_xor(t, off, 64);
			v[0] = t;
		} else {
#pragma unroll
			for (int i = 0; i < N; i++) {
				float t = 0.0f;
#pragma unroll
				for (int w = 0; w < GROUP / 64; w++) t += red[w * N + i];
				v[i] = t;
			}
		}
	}
}

// ---- forward ---------------------------------------------------------------------------------------

// GROUP threads own R rows at a time, each row in registers: one read, one write, bound by memory (16384 x 4096 89 us,
// 6.0 TB/s; 65536 x 1024 89 and 262144 x 256 90; 8192 x 8192 90 and 4096 x 16384 100; a copy of as much by the library 114). Rows
// of up to 1024 elements take (part of) a wave, so that the sums need no barrier; longer ones a block.
// The weights are asked for together with the rows, to wait once; in the large blocks of long rows after the sums instead and
// one vector after the other, so that 64 registers are enough even for 16 elements a thread and more blocks share a unit
// (16384 x 4096 94 -> 89, 8192 x 8192 98 -> 90, 4096 x 16384 125 -> 100).
template <int GROUP, int E, Access ACCESS, int R>
__global__ __launch_bounds__(GROUP > 256 ? GROUP : 256, GROUP >= 1024 && E == 16 ? 8 : 1) void layer_norm_kernel(const float* x, const float* __restrict__ weight, const float* __restrict__ bias, float* y,
                                                                                float* __restrict__ mean_out, float* __restrict__ rstd_out, size_t rows, int cols, float eps) {
	constexpr int kThreads = GROUP > 256 ? GROUP : 256;
	constexpr bool kLate = GROUP >= 512;
	__shared__ float red[GROUP > 64 ? 2 * R * GROUP / 64 : 1];
	const int lane = threadIdx.x % GROUP;
	const size_t first = ((size_t)blockIdx.x * (kThreads / GROUP) + threadIdx.x / GROUP) * R;
	float v[R][E], sum[R], sq[R];
#pragma unroll
	for (int r = 0; r < R; r++) load_row<GROUP, E, ACCESS>(x + (first + r < rows ? first + r : rows - 1) * cols, v[r], lane, cols);
	float w[E], b[E];
	if constexpr (!kLate) {
		load_shared<GROUP, E, ACCESS>(weight, w, lane, cols, 1.0f);
		load_shared<GROUP, E, ACCESS>(bias, b, lane, cols, 0.0f);
	}
#pragma unroll
	for (int r = 0; r < R; r++) {
		sum[r] = 0.0f;
#pragma unroll
		for (int i = 0; i < E; i++) sum[r] += v[r][i];
	}
	group_sums<GROUP, R>(sum, red);
	const float count = (float)cols;
#pragma unroll
	for (int r = 0; r < R; r++) {
		sum[r] /= count;
		sq[r] = 0.0f;
#pragma unroll
		for (int i = 0; i < E; i++) {
			v[r][i] -= sum[r];
			sq[r] += inside<GROUP, ACCESS>(i, lane, cols) ? v[r][i] * v[r][i] : 0.0f;
		}
	}
	group_sums<GROUP, R>(sq, red + (GROUP > 64 ? R * GROUP / 64 : 0));
#pragma unroll
	for (int r = 0; r < R; r++) {
		if (first + r >= rows) break;
		const float rstd = 1.0f / sqrtf(sq[r] / count + eps);
		if constexpr (kLate) {
			int at = lane;  // the places are worked out anew, not kept over the sums
			asm volatile("" : "+v"(at));
			load_shared<GROUP, E, ACCESS>(weight, w, at, cols, 1.0f);
#pragma unroll
			for (int i = 0; i < E; i++) v[r][i] = v[r][i] * rstd * w[i];
			asm volatile("" : "+v"(at));
			load_shared<GROUP, E, ACCESS>(bias, w, at, cols, 0.0f);
#pragma unroll
			for (int i = 0; i < E; i++) v[r][i] += w[i];
		} else {
#pragma unroll
			for (int i = 0; i < E; i++) v[r][i] = v[r][i] * rstd * w[i] + b[i];
		}
		store_row<GROUP, E, ACCESS, true>(y + (first + r) * cols, v[r], lane, cols);
		if (lane == 0) {
			if (mean_out) mean_out[first + r] = sum[r];
			if (rstd_out) rstd_out[first + r] = rstd;
		}
	}
}

// Rows too long for the registers of a block: cut into segments of kLnSegment. One kernel leaves the sum and the sum
// of squares about its own mean of every segment, a second joins a row's segments,
//   mean = sum n_s mean_s / n,   sum of squares = sum (q_s + n_s (mean_s - mean)^2),
// and normalises one of them: two reads and one write whatever the number of rows (4096 x 16388: 38 + 83 us; the second read
// comes from the last-level cache in part).
constexpr int kLnSegment = 8192, kLnSegmentElements = kLnSegment / kLnThreads;

template <Access ACCESS>
__global__ __launch_bounds__(kLnThreads) void layer_norm_segment_kernel(const float* __restrict__ x, float2* __restrict__ stats, int cols, int segments) {
	__shared__ float red[2 * kLnThreads / 64];
	const size_t row = blockIdx.x / segments;
	const int c0 = (int)(blockIdx.x % segments) * kLnSegment, count = cols - c0 < kLnSegment ? cols - c0 : kLnSegment;
	const float* p = x + row * cols + c0;
	float v[kLnSegmentElements], sum[1] = {0.0f}, sq[1] = {0.0f};
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(p, v, threadIdx.x, count, 0.0f);
#pragma unroll
	for (int i = 0; i < kLnSegmentElements; i++) sum[0] += v[i];
	group_sums<kLnThreads, 1>(sum, red);
	const float mean = sum[0] / (float)count;
#pragma unroll
	for (int i = 0; i < kLnSegmentElements; i++) {
		const float d = v[i] - mean;
		sq[0] += inside<kLnThreads, ACCESS>(i, threadIdx.x, count) ? d * d : 0.0f;
	}
	group_sums<kLnThreads, 1>(sq, red + kLnThreads / 64);
	if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(mean, sq[0]);
}

template <Access ACCESS>
__global__ __launch_bounds__(kLnThreads) void layer_norm_apply_kernel(const float* x, const float* __restrict__ weight, const float* __restrict__ bias, float* y, float* __restrict__ mean_out,
                                                                      float* __restrict__ rstd_out, const float2* __restrict__ stats, int cols, int segments, float eps) {
	__shared__ float red[2 * kLnThreads / 64];
	const size_t row = blockIdx.x / segments;
	const int segment = (int)(blockIdx.x % segments), c0 = segment * kLnSegment, count = cols - c0 < kLnSegment ? cols - c0 : kLnSegment;
	float v[kLnSegmentElements];
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(x + row * cols + c0, v, threadIdx.x, count, 0.0f);
	const float2* st = stats + row * segments;
	float sum[1] = {0.0f}, sq[1] = {0.0f};
	for (int s = threadIdx.x; s < segments; s += kLnThreads) sum[0] += st[s].x * (float)(cols - s * kLnSegment < kLnSegment ? cols - s * kLnSegment : kLnSegment);
	group_sums<kLnThreads, 1>(sum, red);
	const float mean = sum[0] / (float)cols;
	for (int s = threadIdx.x; s < segments; s += kLnThreads) {
		const float d = st[s].x - mean;
		sq[0] += st[s].y + d * d * (float)(cols - s * kLnSegment < kLnSegment ? cols - s * kLnSegment : kLnSegment);
	}
	group_sums<kLnThreads, 1>(sq, red + kLnThreads / 64);
	const float rstd = 1.0f / sqrtf(sq[0] / (float)cols + eps);
	float w[kLnSegmentElements];
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(weight ? weight + c0 : nullptr, w, threadIdx.x, count, 1.0f);
#pragma unroll
	for (int i = 0; i < kLnSegmentElements; i++) v[i] = (v[i] - mean) * rstd * w[i];
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(bias ? bias + c0 : nullptr, w, threadIdx.x, count, 0.0f);
#pragma unroll
	for (int i = 0; i < kLnSegmentElements; i++) v[i] += w[i];
	store_row<kLnThreads, kLnSegmentElements, ACCESS, true>(y + row * cols + c0, v, threadIdx.x, count);
	if (segment == 0 && threadIdx.x == 0) {
		if (mean_out) mean_out[row] = mean;
		if (rstd_out) rstd_out[row] = rstd;
	}
}

// ---- backward --------------------------------------------------------------------------------------

// dw and db of some columns (a power of two up to kLnColumns) from c0 on, by one block that goes through all rows: with few
// rows. That many threads side by side, the others at other rows; the threads' sums are added in a fixed order.
constexpr int kLnColumns = 16;
template <int THREADS>
__device__ __forceinline__ void column_sums(const float* x, const float* dy, const float* __restrict__ mean, const float* __restrict__ rstd, float* __restrict__ dweight, float* __restrict__ dbias,
                                            size_t rows, int cols, int c0, int columns) {
	__shared__ float red[2][THREADS / 64][kLnColumns];
	constexpr int kAhead = 8;
	const int slices = THREADS / columns, mine = threadIdx.x & (columns - 1), c = c0 + mine;
	float dw = 0.0f, db = 0.0f;
	if (c < cols)
		for (size_t r0 = threadIdx.x / columns; r0 < rows; r0 += slices * kAhead) {
			float vx[kAhead], vdy[kAhead], m[kAhead], s[kAhead];
#pragma unroll
			for (int u = 0; u < kAhead; u++) {
				const size_t r = r0 + u * slices < rows ? r0 + u * slices : r0;
				vx[u] = x[r * cols + c];
				vdy[u] = dy[r * cols + c];
				m[u] = mean[r];
				s[u] = rstd[r];
			}
#pragma unroll
			for (int u = 0; u < kAhead; u++) {
				if (r0 + u * slices >= rows) break;
				dw += vdy[u] * ((vx[u] - m[u]) * s[u]);
				db += vdy[u];
			}
		}
	for (int off = columns; off < 64; off *= 2) {
		dw += __shfl_xor(dw, off, 64);
		db += __shfl_xor(db, off, 64);
	}
	const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
	if (lane < columns) {
		red[0][wave][lane] = dw;
		red[1][wave][lane] = db;
	}
	__syncthreads();
	if ((int)threadIdx.x < 2 * columns) {
		const int which = (int)threadIdx.x >= columns;
		float t = 0.0f;
#pragma unroll
		for (int w = 0; w < THREADS / 64; w++) t += red[which][w][mine];
		float* to = which ? dbias : dweight;
		if (to && c < cols) to[c] = t;
	}
}

// As the forward kernel, but a group stays and takes rows in turn (`step` groups in all): the column sums of dy xhat and
// dy of its rows stay in its registers and leave once, partial[block][2][cols], after the groups of a block have added
// theirs up in group memory. Each of x and dy is read once, dx written once: bound by memory (262144 x 256 131 us, 6.1 TB/s;
// 16384 x 4096 133; 65536 x 1024 135; 4096 x 16384 145), and the fold behind it takes 5 us. Blocks from row_blocks on are those
// of column_sums, with few rows; then there is no partial.
template <int GROUP, int E, Access ACCESS, int R>
__global__ __launch_bounds__(GROUP > 256 ? GROUP : 256) void layer_norm_backward_kernel(const float* x, const float* dy, const float* __restrict__ weight, const float* __restrict__ mean,
                                                                                        const float* __restrict__ rstd, float* dx, float* __restrict__ partial, size_t rows, int cols,
                                                                                        unsigned row_blocks, int columns, float* __restrict__ dweight, float* __restrict__ dbias) {
	constexpr int kThreads = GROUP > 256 ? GROUP : 256, kGroups = kThreads / GROUP;
	if (blockIdx.x >= row_blocks) {
		column_sums<kThreads>(x, dy, mean, rstd, dweight, dbias, rows, cols, (blockIdx.x - row_blocks) * columns, columns);
		return;
	}
	// for the sums of a large group (two in turn, so that one barrier a row is enough), then for the join of the groups' columns
	__shared__ float red[GROUP > 64 ? 4 * R * GROUP / 64 : kGroups * GROUP * E];
	const int lane = threadIdx.x % GROUP, group = threadIdx.x / GROUP;
	float w[E], sum_dw[E], sum_db[E];
	load_shared<GROUP, E, ACCESS>(weight, w, lane, cols, 1.0f);
#pragma unroll
	for (int i = 0; i < E; i++) sum_dw[i] = sum_db[i] = 0.0f;
	const size_t step = (size_t)row_blocks * kGroups * R;
	const float count = (float)cols;
	int turn = 0;
	for (size_t first = ((size_t)blockIdx.x * kGroups + group) * R; first < rows; first += step) {
		float vx[R][E], vdy[R][E], m[R], s[R], sums[2 * R];
#pragma unroll
		for (int r = 0; r < R; r++) {
			const size_t row = first + r < rows ? first + r : rows - 1;
			m[r] = mean[row];
			s[r] = rstd[row];
			load_row<GROUP, E, ACCESS>(x + row * cols, vx[r], lane, cols);
			load_row<GROUP, E, ACCESS>(dy + row * cols, vdy[r], lane, cols);
		}
#pragma unroll
		for (int r = 0; r < R; r++) {
			sums[2 * r] = sums[2 * r + 1] = 0.0f;
			const bool real = R == 1 || first + r < rows;
#pragma unroll
			for (int i = 0; i < E; i++) {
				vx[r][i] = (vx[r][i] - m[r]) * s[r];  // xhat; beyond the row dy is 0, and 0 times a finite number adds nothing
				if (!inside<GROUP, ACCESS>(i, lane, cols)) vx[r][i] = 0.0f;
				if (real) {
					sum_dw[i] += vdy[r][i] * vx[r][i];
					sum_db[i] += vdy[r][i];
				}
				vdy[r][i] *= w[i];
				sums[2 * r] += vdy[r][i];
				sums[2 * r + 1] += vdy[r][i] * vx[r][i];
			}
		}
		if (dx) {
			group_sums<GROUP, 2 * R>(sums, red + (GROUP > 64 ? turn * 2 * R * GROUP / 64 : 0));
			turn ^= 1;
#pragma unroll
			for (int r = 0; r < R; r++) {
				if (first + r >= rows) break;
				const float mg = sums[2 * r] / count, mgx = sums[2 * r + 1] / count;
#pragma unroll
				for (int i = 0; i < E; i++) vdy[r][i] = s[r] * (vdy[r][i] - mg - vx[r][i] * mgx);
				// lines that single floats fill in parts are put together in the caches (65536 x 1023 142 us, 157 past them; the forward
				// pass gains from it in some shapes and loses in others: 16384 x 4095 110 | 116, 4099 x 1001 8.2 | 7.6)
				store_row<GROUP, E, ACCESS, ACCESS != Access::Single>(dx + (first + r) * cols, vdy[r], lane, cols);
			}
		}
	}
	if (!partial) return;
	partial += (size_t)blockIdx.x * 2 * cols;
	if constexpr (kGroups > 1) {
#pragma unroll
		for (int which = 0; which < 2; which++) {
			__syncthreads();
#pragma unroll
			for (int i = 0; i < E; i++) red[(group * E + i) * GROUP + lane] = which ? sum_db[i] : sum_dw[i];
			__syncthreads();
			if (group == 0) {
#pragma unroll
				for (int i = 0; i < E; i++) {
					float t = red[i * GROUP + lane];
					for (int g = 1; g < kGroups; g++) t += red[(g * E + i) * GROUP + lane];
					if (which)
						sum_db[i] = t;
					else
						sum_dw[i] = t;
				}
			}
		}
		if (group != 0) return;
	}
	store_row<GROUP, E, ACCESS, false>(partial, sum_dw, lane, cols);
	store_row<GROUP, E, ACCESS, false>(partial + cols, sum_db, lane, cols);
}

// dx of rows cut into segments: the two sums of every segment, then the join and dx of one segment. A thread writes only
// elements that it alone reads, after reading them. (4096 x 16388: column sums 101, these 86 and 140 us: x and dy are read three
// times. A row of 16384 in registers takes 151 in all, so rows stay there as long as they fit.)
template <Access ACCESS>
__global__ __launch_bounds__(kLnThreads) void layer_norm_segment_sums_kernel(const float* __restrict__ x, const float* __restrict__ dy, const float* __restrict__ weight,
                                                                             const float* __restrict__ mean, const float* __restrict__ rstd, float2* __restrict__ stats, int cols, int segments) {
	__shared__ float red[2 * kLnThreads / 64];
	const size_t row = blockIdx.x / segments;
	const int c0 = (int)(blockIdx.x % segments) * kLnSegment, count = cols - c0 < kLnSegment ? cols - c0 : kLnSegment;
	const float m = mean[row], s = rstd[row];
	float sums[2] = {0.0f, 0.0f};
	float vx[kLnSegmentElements], vdy[kLnSegmentElements], w[kLnSegmentElements];
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(x + row * cols + c0, vx, threadIdx.x, count, 0.0f);
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(dy + row * cols + c0, vdy, threadIdx.x, count, 0.0f);
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(weight ? weight + c0 : nullptr, w, threadIdx.x, count, 1.0f);
#pragma unroll
	for (int i = 0; i < kLnSegmentElements; i++) {
		const float g = vdy[i] * w[i];
		sums[0] += g;
		sums[1] += inside<kLnThreads, ACCESS>(i, threadIdx.x, count) ? g * ((vx[i] - m) * s) : 0.0f;
	}
	group_sums<kLnThreads, 2>(sums, red);
	if (threadIdx.x == 0) stats[blockIdx.x] = make_float2(sums[0], sums[1]);
}

template <Access ACCESS>
__global__ __launch_bounds__(kLnThreads) void layer_norm_segment_dx_kernel(const float* x, const float* dy, const float* __restrict__ weight, const float* __restrict__ mean,
                                                                           const float* __restrict__ rstd, float* dx, const float2* __restrict__ stats, int cols, int segments) {
	__shared__ float red[2 * kLnThreads / 64];
	const size_t row = blockIdx.x / segments;
	const int c0 = (int)(blockIdx.x % segments) * kLnSegment, count = cols - c0 < kLnSegment ? cols - c0 : kLnSegment;
	float vx[kLnSegmentElements], vdy[kLnSegmentElements], w[kLnSegmentElements];
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(x + row * cols + c0, vx, threadIdx.x, count, 0.0f);
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(dy + row * cols + c0, vdy, threadIdx.x, count, 0.0f);
	load_shared<kLnThreads, kLnSegmentElements, ACCESS>(weight ? weight + c0 : nullptr, w, threadIdx.x, count, 1.0f);
	float sums[2] = {0.0f, 0.0f};
	for (int k = threadIdx.x; k < segments; k += kLnThreads) {
		const float2 t = stats[row * segments + k];
		sums[0] += t.x;
		sums[1] += t.y;
	}
	group_sums<kLnThreads, 2>(sums, red);
	const float m = mean[row], s = rstd[row], mg = sums[0] / (float)cols, mgx = sums[1] / (float)cols;
#pragma unroll
	for (int i = 0; i < kLnSegmentElements; i++) vx[i] = s * (vdy[i] * w[i] - mg - (vx[i] - m) * s * mgx);
	store_row<kLnThreads, kLnSegmentElements, ACCESS, true>(dx + row * cols + c0, vx, threadIdx.x, count);
}

// Partial sums of dw and db for such rows: group (tile of 256 VEC columns, slab of rows), VEC columns per thread.
template <int VEC>
__global__ __launch_bounds__(kLnThreads) void layer_norm_dweight_kernel(const float* __restrict__ x, const float* __restrict__ dy, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                        float* __restrict__ partial, size_t rows, size_t cols, size_t rows_per_slab, unsigned col_tiles) {
	typedef std::conditional_t<VEC == 4, LnVec, float> Vec;
	const size_t c = ((size_t)(blockIdx.x % col_tiles) * kLnThreads + threadIdx.x) * VEC;
	const size_t slab = blockIdx.x / col_tiles;
	if (c >= cols) return;
	const size_t r0 = slab * rows_per_slab, r1 = r0 + rows_per_slab < rows ? r0 + rows_per_slab : rows;
	Vec dw = Vec(0.0f), db = Vec(0.0f);
#pragma unroll 8
	for (size_t r = r0; r < r1; r++) {
		const Vec d = *reinterpret_cast<const Vec*>(dy + r * cols + c), v = *reinterpret_cast<const Vec*>(x + r * cols + c);
		dw += d * ((v - mean[r]) * rstd[r]);
		db += d;
	}
	*reinterpret_cast<Vec*>(partial + (slab * 2) * cols + c) = dw;
	*reinterpret_cast<Vec*>(partial + (slab * 2 + 1) * cols + c) = db;
}

// The sum of the partial results, in a fixed order: a block of 16 waves per 64 of the 2 cols columns, wave w the parts
// w, w + 16, ..., then the waves' sums in the order of the waves.
constexpr int kFoldWaves = 16;
__global__ __launch_bounds__(kFoldWaves * 64) void layer_norm_fold_kernel(const float* __restrict__ partial, float* __restrict__ dweight, float* __restrict__ dbias, size_t parts, size_t cols) {
	__shared__ float red[kFoldWaves][64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const size_t width = 2 * cols;
	for (size_t c0 = (size_t)blockIdx.x * 64; c0 < width; c0 += (size_t)gridDim.x * 64) {
		const size_t c = c0 + lane;
		float sum = 0.0f;
		if (c < width) {
			size_t k = wave;
			for (; k + 7 * kFoldWaves < parts; k += 8 * kFoldWaves) {
				float t[8];
#pragma unroll
				for (int u = 0; u < 8; u++) t[u] = partial[(k + u * kFoldWaves) * width + c];
#pragma unroll
				for (int u = 0; u < 8; u++) sum += t[u];
			}
			for (; k < parts; k += kFoldWaves) sum += partial[k * width + c];
		}
		red[wave][lane] = sum;
		__syncthreads();
		if (wave == 0 && c < width) {
#pragma unroll
			for (int w = 1; w < kFoldWaves; w++) sum += red[w][lane];
			float* to = c < cols ? dweight : dbias;
			if (to) to[c < cols ? c : c - cols] = sum;
		}
		__syncthreads();
	}
}

// ---- which kernel ------------------------------------------------------------------------------------

// A row of 16384 in registers takes 100 us forward and 151 backward for 4096 rows, one of 16388 in segments 121 and 335.
constexpr size_t kLnMostInRegisters = 16384;

// Up to so many rows (twice as many narrow ones) the backward pass is one launch: dw and db need only the rows' statistics, which
// are inputs, so other blocks of the same launch sum the columns, and x and dy are read twice; where dx is x or dy, in a launch
// before. us in the kernels, one launch | two, which also wait 3 us for each other: 16 x 1024 3.3 | 7.0, 256 x 1024 4.8 | 8.0, 256 x
// 4096 5 | 10.7, 512 x 256 4.0 | 7.0, 512 x 4096 13.5 | 17.0, 1024 x 64 5.0 | 6.1; beyond, 1037 x 772 11.6 | 8.7, 2048 x 256 11.6 | 7.0.
constexpr size_t kLnNarrow = 256;
constexpr size_t kLnFewRows = 512;

// Calls f with (threads of a row, elements of a thread, rows at a time) as constants: the smallest group that holds the
// row with four elements a thread up to a wave, then more elements, then a block. Several short rows at a time hide the
// exchanges of their sums behind each other. (16384 x 4096 as 512 threads of 8 | 256 of 16: 94 | 96 us forward with the
// weights asked for early in both, 131 | 144 backward.)
template <bool EVEN, class F>
static void with_row_group(size_t cols, F f) {
	using std::integral_constant;
#define TFHIP_LN_CASE(GROUP, E, R) f(integral_constant<int, GROUP>(), integral_constant<int, E>(), integral_constant<Access, EVEN ? Access::Whole : GROUP >= 512 && E == 16 ? Access::Anywhere : Access::Single>(), integral_constant<int, R>())
	if (cols <= 32) TFHIP_LN_CASE(8, 4, 2);
	else if (cols <= 64) TFHIP_LN_CASE(16, 4, 2);
	else if (cols <= 128) TFHIP_LN_CASE(32, 4, 4);
	else if (cols <= 256) TFHIP_LN_CASE(64, 4, 4);
	else if (cols <= 512) TFHIP_LN_CASE(64, 8, 2);
	else if (cols <= 1024) TFHIP_LN_CASE(64, 16, 1);
	else if (cols <= 2048) TFHIP_LN_CASE(256, 8, 1);
	else if (cols <= 4096) TFHIP_LN_CASE(512, 8, 1);
	else if (cols <= 8192) TFHIP_LN_CASE(512, 16, 1);
	else TFHIP_LN_CASE(1024, 16, 1);
#undef TFHIP_LN_CASE
}

static bool aligned16(const void* a, const void* b, const void* c, const void* d) { return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0; }

template <bool EVEN>
static int layer_norm_forward(const float* x, const float* weight, const float* bias, float* y, float* mean, float* rstd, size_t rows, size_t cols, float eps) {
	State& s = state();
	with_row_group<EVEN>(cols, [&](auto group, auto e, auto access, auto r) {
		constexpr int kGroup = decltype(group)::value, kThreads = kGroup > 256 ? kGroup : 256, kRows = kThreads / kGroup * decltype(r)::value;
		// a launch has fewer than 2^32 threads
		constexpr size_t kMost = ((size_t)1 << 31) / kThreads * kRows;
		for (size_t first = 0; first < rows; first += kMost) {
			const size_t count = rows - first < kMost ? rows - first : kMost;
			hipLaunchKernelGGL((layer_norm_kernel<kGroup, decltype(e)::value, decltype(access)::value, decltype(r)::value>), dim3((unsigned)((count + kRows - 1) / kRows)), dim3(kThreads), 0, s.stream,
			                   x + first * cols, weight, bias, y + first * cols, mean ? mean + first : nullptr, rstd ? rstd + first : nullptr, count, (int)cols, eps);
		}
	});
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}

static int launch_fold(const float* partial, float* dweight, float* dbias, size_t parts, size_t cols) {
	const size_t groups = (2 * cols + 63) / 64;
	hipLaunchKernelGGL(layer_norm_fold_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(kFoldWaves * 64), 0, state().stream, partial, dweight, dbias, parts, cols);
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}

template <bool EVEN>
static int layer_norm_backward(const float* x, const float* dy, const float* weight, const float* mean, const float* rstd, float* dx, float* dweight, float* dbias, size_t rows, size_t cols) {
	State& s = state();
	int rc = TFHIP_OK;
	with_row_group<EVEN>(cols, [&](auto group, auto e, auto access, auto r) {
		constexpr int kGroup = decltype(group)::value, kThreads = kGroup > 256 ? kGroup : 256, kRows = kThreads / kGroup * decltype(r)::value;
		// as many blocks as stay resident, 1024 threads a unit
		const size_t most = (size_t)s.compute_units * 1024 / kThreads, want = (rows + kRows - 1) / kRows, blocks = want < most ? want : most;
		// narrow stretches of columns, so that a thread has fewer rows, where the matrix is small enough to be read in such pieces
		// (16 | 4 columns: 512 x 256 6.8 | 4.0 us, 512 x 1024 7.1 | 5.8, 512 x 4096 13 | 26)
		const int columns = rows > 128 && cols <= 1024 ? 4 : kLnColumns;
		auto launch = [&](unsigned row_blocks, unsigned column_blocks, float* partial) {
			if (rc || row_blocks + column_blocks == 0) return;
			hipLaunchKernelGGL((layer_norm_backward_kernel<kGroup, decltype(e)::value, decltype(access)::value, decltype(r)::value>), dim3(row_blocks + column_blocks), dim3(kThreads), 0, s.stream, x,
			                   dy, weight, mean, rstd, dx, partial, rows, (int)cols, row_blocks, columns, dweight, dbias);
			const hipError_t err = hipGetLastError();
			if (err != hipSuccess) rc = fail_hip(err, "layer norm backward launch");
		};
		if (rows <= (cols <= kLnNarrow ? 2 * kLnFewRows : kLnFewRows)) {
			const unsigned row_blocks = dx ? (unsigned)blocks : 0, column_blocks = dweight || dbias ? (unsigned)((cols + columns - 1) / columns) : 0;
			if (dx == x || dx == dy) {  // all columns before the first row is overwritten
				launch(0, column_blocks, nullptr);
				launch(row_blocks, 0, nullptr);
			} else {
				launch(row_blocks, column_blocks, nullptr);
			}
			return;
		}
		float* partial = nullptr;
		if (dweight || dbias) {
			partial = (float*)scratch(blocks * 2 * cols * sizeof(float));
			if (!partial) {
				rc = TFHIP_ERR_HIP;
				return;
			}
		}
		launch((unsigned)blocks, 0, partial);
		if (!rc && partial) rc = launch_fold(partial, dweight, dbias, blocks, cols);
	});
	return rc;
}

template <bool EVEN>
static int layer_norm_long_backward(const float* x, const float* dy, const float* weight, const float* mean, const float* rstd, float* dx, float* dweight, float* dbias, size_t rows, size_t cols) {
	constexpr Access kAccess = EVEN ? Access::Whole : Access::Anywhere;
	constexpr int kVec = EVEN ? 4 : 1;  // columns of a thread in the column sums
	State& s = state();
	const size_t segments = (cols + kLnSegment - 1) / kLnSegment, col_tiles = (cols + kLnThreads * kVec - 1) / (kLnThreads * kVec);
	if (rows * segments > 0xFFFFFF) return fail(TFHIP_ERR_ARG, "layer norm of %zu x %zu is too large", rows, cols);
	size_t slabs = (size_t)s.compute_units * 8 / col_tiles;
	if (slabs > (rows + 15) / 16) slabs = (rows + 15) / 16;
	if (slabs < 1) slabs = 1;
	const size_t per = (rows + slabs - 1) / slabs;
	slabs = (rows + per - 1) / per;
	const size_t stats_bytes = (rows * segments * sizeof(float2) + 255) & ~size_t(255);
	char* base = (char*)scratch(stats_bytes + slabs * 2 * cols * sizeof(float));
	if (!base) return TFHIP_ERR_HIP;
	float2* stats = (float2*)base;
	float* partial = (float*)(base + stats_bytes);
	if (dweight || dbias) {  // before dx, which may overwrite x or dy
		hipLaunchKernelGGL(layer_norm_dweight_kernel<kVec>, dim3((unsigned)(col_tiles * slabs)), dim3(kLnThreads), 0, s.stream, x, dy, mean, rstd, partial, rows, cols, per, (unsigned)col_tiles);
		TFHIP_CHECK_LAUNCH();
		const int rc = launch_fold(partial, dweight, dbias, slabs, cols);
		if (rc) return rc;
	}
	if (dx) {
		const dim3 grid((unsigned)(rows * segments)), block(kLnThreads);
		hipLaunchKernelGGL(layer_norm_segment_sums_kernel<kAccess>, grid, block, 0, s.stream, x, dy, weight, mean, rstd, stats, (int)cols, (int)segments);
		TFHIP_CHECK_LAUNCH();
		hipLaunchKernelGGL(layer_norm_segment_dx_kernel<kAccess>, grid, block, 0, s.stream, x, dy, weight, mean, rstd, dx, (const float2*)stats, (int)cols, (int)segments);
		TFHIP_CHECK_LAUNCH();
	}
	return TFHIP_OK;
}

template <bool EVEN>
static int layer_norm_long_forward(const float* x, const float* weight, const float* bias, float* y, float* mean, float* rstd, size_t rows, size_t cols, float eps) {
	constexpr Access kAccess = EVEN ? Access::Whole : Access::Anywhere;
	State& s = state();
	const size_t segments = (cols + kLnSegment - 1) / kLnSegment;
	if (rows * segments > 0xFFFFFF) return fail(TFHIP_ERR_ARG, "layer norm of %zu x %zu is too large", rows, cols);
	float2* stats = (float2*)scratch(rows * segments * sizeof(float2));
	if (!stats) return TFHIP_ERR_HIP;
	const dim3 grid((unsigned)(rows * segments)), block(kLnThreads);
	hipLaunchKernelGGL(layer_norm_segment_kernel<kAccess>, grid, block, 0, s.stream, x, stats, (int)cols, (int)segments);
	TFHIP_CHECK_LAUNCH();
	hipLaunchKernelGGL(layer_norm_apply_kernel<kAccess>, grid, block, 0, s.stream, x, weight, bias, y, mean, rstd, (const float2*)stats, (int)cols, (int)segments, eps);
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}

static int check_extent(size_t rows, size_t cols) {
	if (cols == 0) return fail(TFHIP_ERR_ARG, "layer norm over rows without columns");
	if (rows > 0x7FFFFFFF || cols > 0x7FFFFFFF) return fail(TFHIP_ERR_ARG, "layer norm of %zu x %zu: a dimension is beyond 2^31 - 1", rows, cols);
	return TFHIP_OK;
}

// Every output against every other buffer of the call; may_equal: the pairs where the whole output may be the input.
struct Range {
	const char* name;
	const void* p;
	size_t words;
	bool output;
	bool may_equal_input;  // of an output: it may be exactly an input of the same size that is so marked
};
static int check_disjoint(const Range* r, int n) {
	for (int a = 0; a < n; a++)
		for (int b = a + 1; b < n; b++) {
			if (!r[a].output && !r[b].output) continue;
			if (!words_overlap(r[a].p, r[a].words, r[b].p, r[b].words)) continue;
			if (r[a].p == r[b].p && r[a].words == r[b].words && r[a].may_equal_input && r[b].may_equal_input && r[a].output != r[b].output) continue;
			return fail(TFHIP_ERR_ARG, "layer norm: %s and %s overlap", r[a].name, r[b].name);
		}
	return TFHIP_OK;
}

}  // namespace tfhip

using namespace tfhip;

extern "C" int tfhip_layer_norm_rows_f32(const float* x, const float* weight, const float* bias, float* y, float* mean, float* rstd, size_t rows, size_t cols, float eps) {
	int rc = check_extent(rows, cols);
	if (rc) return rc;
	if (!(eps >= 0.0f) || !isfinite(eps)) return fail(TFHIP_ERR_ARG, "layer norm with eps = %g: a finite number of at least 0 is needed", (double)eps);
	if (rows == 0) return TFHIP_OK;
	if (!x || !y) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_layer_norm_rows_f32");
	const Range ranges[] = {{"x", x, rows * cols, false, true}, {"weight", weight, cols, false, false}, {"bias", bias, cols, false, false},
	                        {"y", y, rows * cols, true, true},  {"mean", mean, rows, true, false},      {"rstd", rstd, rows, true, false}};
	rc = check_disjoint(ranges, 6);
	if (rc) return rc;
	TFHIP_REQUIRE_INIT();
	TFHIP_HOLD_DEVICE();
	const bool even = cols % 4 == 0 && aligned16(x, y, weight, bias);
	if (cols > kLnMostInRegisters) return (even ? layer_norm_long_forward<true> : layer_norm_long_forward<false>)(x, weight, bias, y, mean, rstd, rows, cols, eps);
	return (even ? layer_norm_forward<true> : layer_norm_forward<false>)(x, weight, bias, y, mean, rstd, rows, cols, eps);
}

extern "C" int tfhip_layer_norm_rows_backward_f32(const float* x, const float* dy, const float* weight, const float* mean, const float* rstd, float* dx, float* dweight, float* dbias, size_t rows,
                                                  size_t cols) {
	int rc = check_extent(rows, cols);
	if (rc) return rc;
	if (!dx && !dweight && !dbias) return fail(TFHIP_ERR_ARG, "tfhip_layer_norm_rows_backward_f32: none of dx, dweight and dbias is wanted");
	if (rows && (!x || !dy || !mean || !rstd)) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_layer_norm_rows_backward_f32");
	const Range ranges[] = {{"x", x, rows * cols, false, true}, {"dy", dy, rows * cols, false, true}, {"weight", weight, cols, false, false},   {"mean", mean, rows, false, false},
	                        {"rstd", rstd, rows, false, false}, {"dx", dx, rows * cols, true, true},  {"dweight", dweight, cols, true, false}, {"dbias", dbias, cols, true, false}};
	rc = check_disjoint(ranges, 8);
	if (rc) return rc;
	TFHIP_REQUIRE_INIT();
	TFHIP_HOLD_DEVICE();
	if (rows == 0) {
		if (dweight && (rc = tfhip_fill_u32(dweight, 0u, cols))) return rc;
		if (dbias && (rc = tfhip_fill_u32(dbias, 0u, cols))) return rc;
		return TFHIP_OK;
	}
	const bool even = cols % 4 == 0 && aligned16(x, dy, weight, dx);
	if (cols > kLnMostInRegisters) return (even ? layer_norm_long_backward<true> : layer_norm_long_backward<false>)(x, dy, weight, mean, rstd, dx, dweight, dbias, rows, cols);
	return (even ? layer_norm_backward<true> : layer_norm_backward<false>)(x, dy, weight, mean, rstd, dx, dweight, dbias, rows, cols);
}
