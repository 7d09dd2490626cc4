// Orthogonalisation of matrices by Newton-Schulz products, as optimisers apply it to the update of a dense layer:
//
//   X = G / (|G|_F + eps);  per step, with its coefficients a, b, c:  A = X X^T,  B = b A + c A^2,  X <- a X + B X
//
// (the transposed form for a matrix with more rows than columns, so that A is the smaller of the two squares). Each
// singular value s of X becomes a s + b s^3 + c s^5. The reference has no such operation; its optimisers stop at the
// element-wise update (Python/TensorFrost/optimizers.py:104-167).

#include "common.h"

#include <math.h>

namespace tfhip {

constexpr int kNsTile = 32;

// Partial sums of squares, in 64 bits: the square of a large fp32 number does not fit fp32.
__global__ __launch_bounds__(256) void ns_norm_kernel(const float* __restrict__ g, double* __restrict__ partial, size_t elements, unsigned parts) {
	__shared__ double red[256];
	const size_t matrix = blockIdx.x / parts, part = blockIdx.x % parts;
	const float* p = g + matrix * elements;
	double sum = 0.0;
	for (size_t i = part * 256 + threadIdx.x; i < elements; i += (size_t)parts * 256) sum += (double)p[i] * (double)p[i];
	red[threadIdx.x] = sum;
	__syncthreads();
	for (int off = 128; off >= 1; off >>= 1) {
		if ((int)threadIdx.x < off) red[threadIdx.x] += red[threadIdx.x + off];
		__syncthreads();
	}
	if (threadIdx.x == 0) partial[blockIdx.x] = red[0];
}

// x = g / (norm + eps), x with at most as many rows as columns (transposed: g is [n, m]).
__global__ __launch_bounds__(256) void ns_scale_kernel(const float* __restrict__ g, const double* __restrict__ partial, unsigned parts, float* __restrict__ x, size_t m, size_t n, bool transposed,
                                                       float eps, unsigned groups) {
	const size_t matrix = blockIdx.x / groups;
	double sum = 0.0;
	for (unsigned k = 0; k < parts; k++) sum += partial[matrix * parts + k];
	const double norm = sqrt(sum) + (double)eps;
	const float r = !isfinite(norm) ? nanf("") : norm > 0.0 ? (float)(1.0 / norm) : 0.0f;
	for (size_t i = (size_t)(blockIdx.x % groups) * 256 + threadIdx.x; i < m * n; i += (size_t)groups * 256) {
		const size_t row = i / n, col = i % n;
		x[matrix * m * n + i] = r * (transposed ? g[matrix * m * n + col * m + row] : g[matrix * m * n + i]);
	}
}

// C = alpha P op(Q) + beta D, fp32, a 32 x 32 tile per group of 256 threads. P [M, K]; Q [N, K] (nt) or [K, N].
template <bool NT>
__global__ __launch_bounds__(256) void ns_product_kernel(const float* __restrict__ P, const float* __restrict__ Q, const float* __restrict__ D, float* __restrict__ C, size_t M, size_t N, size_t K,
                                                         float alpha, float beta) {
	__shared__ float p[kNsTile][kNsTile + 1], q[kNsTile][kNsTile + 1];
	P += blockIdx.z * M * K;
	Q += blockIdx.z * N * K;
	D += blockIdx.z * M * N;
	C += blockIdx.z * M * N;
	const size_t m0 = (size_t)blockIdx.y * kNsTile, n0 = (size_t)blockIdx.x * kNsTile;
	const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
	float acc[4] = {};
	for (size_t k0 = 0; k0 < K; k0 += kNsTile) {
		for (int i = ty; i < kNsTile; i += 8) {
			p[i][tx] = m0 + i < M && k0 + tx < K ? P[(m0 + i) * K + k0 + tx] : 0.0f;
			if (NT)
				q[i][tx] = n0 + i < N && k0 + tx < K ? Q[(n0 + i) * K + k0 + tx] : 0.0f;
			else
				q[tx][i] = n0 + tx < N && k0 + i < K ? Q[(k0 + i) * N + n0 + tx] : 0.0f;
		}
		__syncthreads();
		for (int k = 0; k < kNsTile; k++)
#pragma unroll
			for (int j = 0; j < 4; j++) acc[j] += p[ty + 8 * j][k] * q[tx][k];
		__syncthreads();
	}
#pragma unroll
	for (int j = 0; j < 4; j++) {
		const size_t row = m0 + ty + 8 * j, col = n0 + tx;
		if (row < M && col < N) C[row * N + col] = alpha * acc[j] + (beta != 0.0f ? beta * D[row * N + col] : 0.0f);
	}
}

__global__ __launch_bounds__(256) void ns_store_kernel(const float* __restrict__ x, float* __restrict__ out, size_t m, size_t n, bool transposed, unsigned groups) {
	const size_t matrix = blockIdx.x / groups;
	for (size_t i = (size_t)(blockIdx.x % groups) * 256 + threadIdx.x; i < m * n; i += (size_t)groups * 256) {
		const size_t row = i / n, col = i % n;
		out[matrix * m * n + (transposed ? col * m + row : i)] = x[matrix * m * n + i];
	}
}

}  // namespace tfhip

using namespace tfhip;

extern "C" int tfhip_newton_schulz_f32(const float* g, float* out, size_t batch, size_t rows, size_t cols, int steps, const float* coefficients, float eps) {
	if (rows == 0 || cols == 0) return fail(TFHIP_ERR_ARG, "orthogonalisation of an empty matrix (%zu x %zu)", rows, cols);
	if (rows > 32768 || cols > 0x7FFFFF || cols * rows > 0x7FFFFFFF) {
		if (cols > 32768 || rows > 0x7FFFFF || cols * rows > 0x7FFFFFFF)
			return fail(TFHIP_ERR_ARG, "orthogonalisation of a %zu x %zu matrix: at most 32768 on its shorter side and 2^31 - 1 elements", rows, cols);
	}
	if (batch > 65535) return fail(TFHIP_ERR_ARG, "more than 65535 matrices in one batch (%zu)", batch);
	if (steps < 1 || steps > 64) return fail(TFHIP_ERR_ARG, "%d Newton-Schulz steps (1 to 64 are taken)", steps);
	if (!coefficients) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_newton_schulz_f32");
	for (int i = 0; i < 3 * steps; i++)
		if (!isfinite(coefficients[i])) return fail(TFHIP_ERR_ARG, "coefficient %d of the Newton-Schulz steps is not finite", i);
	if (!(eps >= 0.0f) || !isfinite(eps)) return fail(TFHIP_ERR_ARG, "Newton-Schulz with eps = %g: a finite number of at least 0 is needed", (double)eps);
	if (batch == 0) return TFHIP_OK;
	if (!g || !out) return fail(TFHIP_ERR_ARG, "null pointer passed to tfhip_newton_schulz_f32");
	const size_t elements = rows * cols;
	if (g != out && words_overlap(g, batch * elements, out, batch * elements)) return fail(TFHIP_ERR_ARG, "Newton-Schulz: g and out overlap without being the same");
	TFHIP_REQUIRE_INIT();
	TFHIP_HOLD_DEVICE();
	State& s = state();
	const bool transposed = rows > cols;
	const size_t m = transposed ? cols : rows, n = transposed ? rows : cols;
	const unsigned parts = (unsigned)(elements < 4096 ? 1 : elements / 4096 < 256 ? elements / 4096 : 256);
	const size_t norm_bytes = (batch * parts * sizeof(double) + 255) & ~size_t(255);
	const size_t x_bytes = (batch * elements * sizeof(float) + 255) & ~size_t(255), a_bytes = (batch * m * m * sizeof(float) + 255) & ~size_t(255);
	char* base = (char*)scratch(norm_bytes + 2 * x_bytes + 2 * a_bytes);
	if (!base) return TFHIP_ERR_HIP;
	double* partial = (double*)base;
	float* x = (float*)(base + norm_bytes);
	float* x2 = (float*)(base + norm_bytes + x_bytes);
	float* A = (float*)(base + norm_bytes + 2 * x_bytes);
	float* B = (float*)(base + norm_bytes + 2 * x_bytes + a_bytes);
	const unsigned groups = (unsigned)(elements / 1024 + 1 < 1024 ? elements / 1024 + 1 : 1024);
	hipLaunchKernelGGL(ns_norm_kernel, dim3((unsigned)batch * parts), dim3(256), 0, s.stream, g, partial, elements, parts);
	TFHIP_CHECK_LAUNCH();
	hipLaunchKernelGGL(ns_scale_kernel, dim3((unsigned)batch * groups), dim3(256), 0, s.stream, g, (const double*)partial, parts, x, m, n, transposed, eps, groups);
	TFHIP_CHECK_LAUNCH();
	const unsigned mt = (unsigned)((m + kNsTile - 1) / kNsTile), nt = (unsigned)((n + kNsTile - 1) / kNsTile);
	for (int k = 0; k < steps; k++) {
		const float a = coefficients[3 * k], b = coefficients[3 * k + 1], c = coefficients[3 * k + 2];
		hipLaunchKernelGGL(ns_product_kernel<true>, dim3(mt, mt, (unsigned)batch), dim3(256), 0, s.stream, x, x, A, A, m, m, n, 1.0f, 0.0f);
		TFHIP_CHECK_LAUNCH();
		hipLaunchKernelGGL(ns_product_kernel<true>, dim3(mt, mt, (unsigned)batch), dim3(256), 0, s.stream, A, A, A, B, m, m, m, c, b);
		TFHIP_CHECK_LAUNCH();
		hipLaunchKernelGGL(ns_product_kernel<false>, dim3(nt, mt, (unsigned)batch), dim3(256), 0, s.stream, B, x, x, x2, m, n, m, 1.0f, a);
		TFHIP_CHECK_LAUNCH();
		float* t = x;
		x = x2;
		x2 = t;
	}
	hipLaunchKernelGGL(ns_store_kernel, dim3((unsigned)batch * groups), dim3(256), 0, s.stream, (const float*)x, out, m, n, transposed, groups);
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}
