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

namespace tfhip {

constexpr int kLnThreads = 256;

// The sum of v over the group, in every thread. `red` holds one float per wave.
template <int THREADS>
__device__ __forceinline__ float group_sum(float v, float* red) {
	v = wave_reduce(v, OpSum());
	__syncthreads();
	if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
	__syncthreads();
	float t = 0.0f;
#pragma unroll
	for (int w = 0; w < THREADS / 64; w++) t += red[w];
	return t;
}

// A group per row, the row read three times (from the caches after the first).
__global__ __launch_bounds__(kLnThreads) void layer_norm_long_kernel(const float* x, const float* __restrict__ weight, const float* __restrict__ bias, float* y, float* __restrict__ mean_out,
                                                                     float* __restrict__ rstd_out, size_t rows, size_t cols, float eps) {
	__shared__ float red[kLnThreads / 64];
	for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
		const float* px = x + row * cols;
		float* py = y + row * cols;
		float sum = 0.0f;
		for (size_t c = threadIdx.x; c < cols; c += kLnThreads) sum += px[c];
		const float mean = group_sum<kLnThreads>(sum, red) / (float)cols;
		float sq = 0.0f;
		for (size_t c = threadIdx.x; c < cols; c += kLnThreads) {
			const float d = px[c] - mean;
			sq += d * d;
		}
		const float rstd = 1.0f / sqrtf(group_sum<kLnThreads>(sq, red) / (float)cols + eps);
		for (size_t c = threadIdx.x; c < cols; c += kLnThreads) py[c] = (px[c] - mean) * rstd * (weight ? weight[c] : 1.0f) + (bias ? bias[c] : 0.0f);
		if (threadIdx.x == 0) {
			if (mean_out) mean_out[row] = mean;
			if (rstd_out) rstd_out[row] = rstd;
		}
	}
}

// dx: a group per row, the row of x and of dy read twice. A thread writes only elements it has read, after the sums:
// dx may be x or dy.
__global__ __launch_bounds__(kLnThreads) void layer_norm_long_dx_kernel(const float* x, const float* dy, const float* __restrict__ weight, const float* __restrict__ mean,
                                                                        const float* __restrict__ rstd, float* dx, size_t rows, size_t cols) {
	__shared__ float red[kLnThreads / 64];
	for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
		const size_t at = row * cols;
		const float m = mean[row], s = rstd[row];
		float sum_g = 0.0f, sum_gx = 0.0f;
		for (size_t c = threadIdx.x; c < cols; c += kLnThreads) {
			const float g = dy[at + c] * (weight ? weight[c] : 1.0f);
			sum_g += g;
			sum_gx += g * ((x[at + c] - m) * s);
		}
		const float mean_g = group_sum<kLnThreads>(sum_g, red) / (float)cols;
		const float mean_gx = group_sum<kLnThreads>(sum_gx, red) / (float)cols;
		for (size_t c = threadIdx.x; c < cols; c += kLnThreads) {
			const float g = dy[at + c] * (weight ? weight[c] : 1.0f);
			const float xhat = (x[at + c] - m) * s;
			dx[at + c] = s * (g - mean_g - xhat * mean_gx);
		}
	}
}

// Partial sums of dw and db: group (tile of 256 columns, slab of rows), one column per thread. partial[slab][2][cols].
__global__ __launch_bounds__(kLnThreads) void layer_norm_dweight_kernel(const float* __restrict__ x, const float* __restrict__ dy, const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                        float* __restrict__ partial, size_t rows, size_t cols, size_t rows_per_slab, unsigned col_tiles) {
	const size_t c = (size_t)(blockIdx.x % col_tiles) * kLnThreads + threadIdx.x;
	const size_t slab = blockIdx.x / col_tiles;
	if (c >= cols) return;
	const size_t r0 = slab * rows_per_slab, r1 = r0 + rows_per_slab < rows ? r0 + rows_per_slab : rows;
	float dw = 0.0f, db = 0.0f;
	for (size_t r = r0; r < r1; r++) {
		const float d = dy[r * cols + c];
		dw += d * ((x[r * cols + c] - mean[r]) * rstd[r]);
		db += d;
	}
	partial[(slab * 2) * cols + c] = dw;
	partial[(slab * 2 + 1) * cols + c] = db;
}

__global__ __launch_bounds__(kLnThreads) void layer_norm_fold_kernel(const float* __restrict__ partial, float* __restrict__ dweight, float* __restrict__ dbias, size_t slabs, size_t cols) {
	const size_t c = (size_t)blockIdx.x * kLnThreads + threadIdx.x;
	if (c >= cols) return;
	float dw = 0.0f, db = 0.0f;
	for (size_t k = 0; k < slabs; k++) {
		dw += partial[(k * 2) * cols + c];
		db += partial[(k * 2 + 1) * cols + c];
	}
	if (dweight) dweight[c] = dw;
	if (dbias) dbias[c] = db;
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
	State& s = state();
	const size_t groups = rows < 65536 ? rows : 65536;
	hipLaunchKernelGGL(layer_norm_long_kernel, dim3((unsigned)groups), dim3(kLnThreads), 0, s.stream, x, weight, bias, y, mean, rstd, rows, cols, eps);
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
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
	State& s = state();
	if (rows == 0) {
		if (dweight && (rc = tfhip_fill_u32(dweight, 0u, cols))) return rc;
		if (dbias && (rc = tfhip_fill_u32(dbias, 0u, cols))) return rc;
		return TFHIP_OK;
	}
	if (dweight || dbias) {  // before dx, which may overwrite x or dy
		const size_t col_tiles = (cols + kLnThreads - 1) / kLnThreads;
		size_t slabs = (size_t)s.compute_units * 8 / col_tiles;
		if (slabs > (rows + 15) / 16) slabs = (rows + 15) / 16;
		if (slabs < 1) slabs = 1;
		const size_t per = (rows + slabs - 1) / slabs;
		slabs = (rows + per - 1) / per;
		float* partial = (float*)scratch(slabs * 2 * cols * sizeof(float));
		if (!partial) return TFHIP_ERR_HIP;
		hipLaunchKernelGGL(layer_norm_dweight_kernel, dim3((unsigned)(col_tiles * slabs)), dim3(kLnThreads), 0, s.stream, x, dy, mean, rstd, partial, rows, cols, per, (unsigned)col_tiles);
		TFHIP_CHECK_LAUNCH();
		hipLaunchKernelGGL(layer_norm_fold_kernel, dim3((unsigned)col_tiles), dim3(kLnThreads), 0, s.stream, (const float*)partial, dweight, dbias, slabs, cols);
		TFHIP_CHECK_LAUNCH();
	}
	if (dx) {
		const size_t groups = rows < 65536 ? rows : 65536;
		hipLaunchKernelGGL(layer_norm_long_dx_kernel, dim3((unsigned)groups), dim3(kLnThreads), 0, s.stream, x, dy, weight, mean, rstd, dx, rows, cols);
		TFHIP_CHECK_LAUNCH();
	}
	return TFHIP_OK;
}
