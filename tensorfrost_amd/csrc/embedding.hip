// Embedding lookup with scaling, and the gradient of its table.
//
//   out[i, :] = scale * table[tokens[i], :]            (zeros where tokens[i] lies outside [0, vocab))
//   dtable[v, :] = scale * sum over i with tokens[i] == v of dy[i, :], every row of dtable written
//
// In the reference this is a load with a computed index (TensorFrost/Compiler/Implementations.cpp:451-488 shows the
// remaps) and, backward, an atomic scatter-add of floats, whose result changes with the order in which the adds land.
// Here the positions are sorted by token first (stable), so each row of the gradient is a sum in the order of the
// positions and comes out the same every time.

#include "common.h"

namespace tfhip {

__global__ __launch_bounds__(256) void embedding_kernel(const int32_t* __restrict__ tokens, const float* __restrict__ table, float* __restrict__ out, size_t n, size_t vocab, size_t cols,
                                                        float scale) {
	const int lane = threadIdx.x & 63;
	const size_t waves = (size_t)gridDim.x * 4;
	for (size_t i = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += waves) {
		const int32_t t = tokens[i];
		const bool known = t >= 0 && (size_t)t < vocab;
		const float* src = table + (known ? (size_t)t : 0) * cols;
		for (size_t c = lane; c < cols; c += 64) out[i * cols + c] = known ? scale * src[c] : 0.0f;
	}
}

// keys[i] = the token, or vocab for positions that belong to no row; order[i] = i.
__global__ __launch_bounds__(256) void embedding_keys_kernel(const int32_t* __restrict__ tokens, uint32_t* __restrict__ keys, uint32_t* __restrict__ order, uint32_t n, uint32_t vocab) {
	const uint32_t i = blockIdx.x * 256 + threadIdx.x;
	if (i >= n) return;
	const int32_t t = tokens[i];
	keys[i] = t >= 0 && (uint32_t)t < vocab ? (uint32_t)t : vocab;
	order[i] = i;
}

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

// A wave per row of the table.
__global__ __launch_bounds__(256) void embedding_rows_sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ order, const float* __restrict__ dy, float* __restrict__ dtable,
                                                                 uint32_t n, uint32_t vocab, size_t cols, float scale) {
	const int lane = threadIdx.x & 63;
	const uint32_t waves = gridDim.x * 4;
	for (uint32_t v = blockIdx.x * 4 + (threadIdx.x >> 6); v < vocab; v += waves) {
		const uint32_t first = first_at_least(keys, n, v), last = first_at_least(keys, n, v + 1);
		for (size_t c = lane; c < cols; c += 64) {
			float sum = 0.0f;
			for (uint32_t p = first; p < last; p++) sum += dy[(size_t)order[p] * cols + c];
			dtable[(size_t)v * cols + c] = scale * sum;
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
	size_t groups = (n + 3) / 4;
	if (groups > 65536) groups = 65536;
	hipLaunchKernelGGL(embedding_kernel, dim3((unsigned)groups), dim3(256), 0, s.stream, tokens, table, out, n, vocab, cols, scale);
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
	// The sort takes its status words from the front of the arena: the six arrays lie behind them.
	const size_t words = (n + 63) & ~size_t(63);
	const size_t sort_bytes = radix_sort_scratch_bytes(n);
	char* base = (char*)scratch(sort_bytes + 6 * words * sizeof(uint32_t));
	if (!base) return TFHIP_ERR_HIP;
	uint32_t* a = (uint32_t*)(base + sort_bytes);
	hipLaunchKernelGGL(embedding_keys_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s.stream, tokens, a, a + words, (uint32_t)n, (uint32_t)vocab);
	TFHIP_CHECK_LAUNCH();
	rc = tfhip_radix_sort_kv_u32(a, a + words, a + 2 * words, a + 3 * words, a + 4 * words, a + 5 * words, n);
	if (rc) return rc;
	size_t groups = (vocab + 3) / 4;
	if (groups > 65536) groups = 65536;
	hipLaunchKernelGGL(embedding_rows_sum_kernel, dim3((unsigned)groups), dim3(256), 0, s.stream, (const uint32_t*)(a + 2 * words), (const uint32_t*)(a + 3 * words), dy, dtable, (uint32_t)n,
	                   (uint32_t)vocab, cols, scale);
	TFHIP_CHECK_LAUNCH();
	return TFHIP_OK;
}
