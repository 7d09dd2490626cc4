// TFHipBuffer, HipMemoryManager, HipKernelManager (see HIP.h). Device work goes through the C ABI of libtfhip.
#include <cstdio>

#include "HIP.h"

#include <cctype>
#include <cstring>
#include <cstdlib>
#include <stdexcept>

namespace TFSHIM_NAMESPACE {

using tfhip::DimExpr;

static void Check(int status, const std::string& what) {
	if (status != TFHIP_OK) throw std::runtime_error(what + ": " + tfhip_last_error());
}

// ---- buffers and the memory manager ---------------------------------------------------------------------------

static void ThrowOnError(int status, const char* what) {
	if (status != TFHIP_OK) throw std::runtime_error(std::string(what) + ": " + tfhip_last_error());
}

TFHipBuffer::TFHipBuffer(size_t size) : TFBufferTemplate(size) { ThrowOnError(tfhip_malloc(&device, size), "Failed to allocate device buffer"); }

TFHipBuffer::~TFHipBuffer() {
	if (device) tfhip_free(device);
}

void TFHipBuffer::SetDataAtOffset(size_t offset, const std::vector<uint32_t>& data) {
	if (offset + data.size() > size) throw std::runtime_error("SetDataAtOffset: write of " + std::to_string(data.size()) + " words at " + std::to_string(offset) + " exceeds buffer of " + std::to_string(size));
	ThrowOnError(tfhip_h2d(device, offset, data.data(), data.size()), "Failed to upload data");
}

void TFHipBuffer::GetDataAtOffset(size_t offset, size_t count, uint32_t* data) {
	if (offset + count > size) throw std::runtime_error("GetDataAtOffset: read of " + std::to_string(count) + " words at " + std::to_string(offset) + " exceeds buffer of " + std::to_string(size));
	ThrowOnError(tfhip_d2h(data, device, offset, count), "Failed to read data back");
}

TFBuffer* HipMemoryManager::CreateBuffer(size_t size) {
	TFHipBuffer* buffer = new TFHipBuffer(size);
	owned.insert(buffer);
	return buffer;
}

void HipMemoryManager::DeleteBuffer(TFBuffer* buffer) {
	owned.erase((TFHipBuffer*)buffer);
	delete (TFHipBuffer*)buffer;
}

HipMemoryManager::~HipMemoryManager() {
	for (TFHipBuffer* buffer : owned) delete buffer;
}

// ---- kernels --------------------------------------------------------------------------------------------------

// `text` with every identifier that starts with `from` (followed by anything but a digit: kernel_5, kernel_5_vars,
// kernel_5_s, not kernel_50) starting with `to` instead.
static std::string RenameKernel(const std::string& text, const std::string& from, const std::string& to) {
	std::string out;
	out.reserve(text.size() + 64);
	size_t at = 0;
	while (true) {
		const size_t hit = text.find(from, at);
		if (hit == std::string::npos) break;
		const char before = hit > 0 ? text[hit - 1] : ' ';
		const char after = hit + from.size() < text.size() ? text[hit + from.size()] : ' ';
		const bool whole = !(isalnum((unsigned char)before) || before == '_') && !isdigit((unsigned char)after);
		out.append(text, at, hit - at);
		out += whole ? to : from;
		at = hit + from.size();
	}
	out.append(text, at, std::string::npos);
	return out;
}

void HipKernelManager::CompileKernel(Kernel* kernel) {
	const HipKernelInfo* info = FindKernelInfo(kernel->kernel_id_);
	if (info == nullptr) throw std::runtime_error("Kernel " + std::to_string(kernel->kernel_id_) + " was not generated by the HIP code generator");
	if (!info->primitive.empty()) return;  // served by a precompiled primitive
	// The compiler sees the kernel under a name made from its own text, not under its number: kernel numbers count up
	// with every program a process compiles, so the same kernel compiled again (the same program once more, in another
	// order, in another process) would otherwise never find its code object in the cache. The name is also what a
	// profiler shows, the same from run to run.
	const std::string& numbered = kernel->kernel_name_;
	const std::string anonymous = RenameKernel(kernel->full_generated_code_, numbered, "tfk");
	uint64_t hash = 1469598103934665603ull;
	for (unsigned char c : anonymous) hash = (hash ^ c) * 1099511628211ull;
	char hex[20];
	snprintf(hex, sizeof(hex), "%016llx", (unsigned long long)hash);
	const std::string stable = std::string("tfk_") + hex;
	const std::string source = RenameKernel(kernel->full_generated_code_, numbered, stable);
	tfhip_kernel_t handle = nullptr;
	int status = tfhip_module_compile(source.c_str(), stable.c_str(), compile_options.c_str(), &handle);
	if (status != TFHIP_OK) {
		// Same content as the GL backend's message: which kernel, the compiler's output, then the source
		// (Backends/OpenGL/KernelManager.h:79-83).
		throw std::runtime_error("Error compiling kernel " + std::to_string(kernel->kernel_id_) + "\n" + tfhip_last_error() + "\n" + kernel->full_generated_code_);
	}
	kernel_handles[kernel->kernel_id_] = handle;
	if (!info->scalar_entry.empty()) {
		tfhip_kernel_t scalar = nullptr;
		Check(tfhip_module_get_kernel(handle, RenameKernel(info->scalar_entry, numbered, stable).c_str(), &scalar), "Error loading kernel " + info->scalar_entry);
		scalar_handles[kernel->kernel_id_] = scalar;
	}
	if (!info->batch_entry.empty()) {
		tfhip_kernel_t batched = nullptr;
		Check(tfhip_module_get_kernel(handle, RenameKernel(info->batch_entry, numbered, stable).c_str(), &batched), "Error loading kernel " + info->batch_entry);
		batch_handles[kernel->kernel_id_] = batched;
	}
}

// Kernels that stand for a whole reduction / scan / matmul / sort go to the hand-written primitives.
static void DispatchPrimitive(const HipKernelInfo* kernel, const TFDispatchInfo& info) {
	const std::string& p = kernel->primitive;
	const size_t n_tensors = info.read_write_count + info.read_only_count;
	if (n_tensors != kernel->primitive_tensors || info.variable_count != kernel->primitive_variables + 1)
		throw std::runtime_error("Primitive " + p + " expects " + std::to_string(kernel->primitive_tensors) + " tensors and " +
		                         std::to_string(kernel->primitive_variables) + " variables");
	auto buf = [&](size_t i) -> void* {
		const TFTensor& t = i < info.read_write_count ? info.read_write_tensors[i] : info.read_only_tensors[i - info.read_write_count];
		return ((TFHipBuffer*)t.buffer)->GetNative();
	};
	auto var = [&](size_t i) { return (size_t)info.variables[i]; };
	auto real = [&](size_t i) {
		float v;
		memcpy(&v, &info.variables[i], sizeof(v));
		return v;
	};
	int status;
	if (p.rfind("sgemm_", 0) == 0) {
		// sgemm_<nn|nt|tn>[_<bias|bias_relu|mask_positive>]
		const std::string layout_name = p.substr(6, 2), tail = p.size() > 9 ? p.substr(9) : "";
		const int layout = layout_name == "nn" ? TFHIP_GEMM_NN : layout_name == "nt" ? TFHIP_GEMM_NT : layout_name == "tn" ? TFHIP_GEMM_TN : -1;
		const int epilogue = tail.empty() ? TFHIP_EPILOGUE_NONE : tail == "bias" ? TFHIP_EPILOGUE_BIAS : tail == "bias_relu" ? TFHIP_EPILOGUE_BIAS_RELU
		                     : tail == "mask_positive" ? TFHIP_EPILOGUE_MASK_POSITIVE : -1;
		if (layout < 0 || epilogue < 0 || n_tensors != (epilogue ? 4u : 3u)) throw std::runtime_error("Unknown primitive " + p);
		status = tfhip_sgemm_fused(layout, (const float*)buf(1), (const float*)buf(2), (float*)buf(0), var(0), var(1), var(2), epilogue,
		                           epilogue ? (const float*)buf(3) : nullptr);
	} else if (p.rfind("reduce_rows_", 0) == 0 || p.rfind("reduce_cols_", 0) == 0) {
		const std::string op = p.substr(12);
		const int code = op == "sum" ? TFHIP_REDUCE_SUM : op == "max" ? TFHIP_REDUCE_MAX : op == "min" ? TFHIP_REDUCE_MIN : -1;
		if (code < 0) throw std::runtime_error("Unknown primitive " + p);
		auto fn = p[7] == 'r' ? tfhip_reduce_rows_f32 : tfhip_reduce_cols_f32;
		status = fn(code, (const float*)buf(1), (float*)buf(0), var(0), var(1));
	} else if (p == "softmax_rows") {
		status = tfhip_softmax_rows_f32((const float*)buf(1), (float*)buf(0), var(0), var(1));
	} else if (p == "scan_u32" || p == "scan_i32") {
		status = tfhip_scan_inclusive_u32((const uint32_t*)buf(1), (uint32_t*)buf(0), var(0));
	} else if (p == "scan_f32") {
		status = tfhip_scan_inclusive_f32((const float*)buf(1), (float*)buf(0), var(0));
	} else if (p.rfind("radix_sort_kv_", 0) == 0) {
		const std::string kind = p.substr(14);
		const int code = kind == "u32" ? TFHIP_KEY_U32 : kind == "i32" ? TFHIP_KEY_I32 : kind == "f32" ? TFHIP_KEY_F32 : -1;
		if (code < 0) throw std::runtime_error("Unknown primitive " + p);
		status = tfhip_radix_sort_kv(code, (const uint32_t*)buf(4), (const uint32_t*)buf(5), (uint32_t*)buf(0), (uint32_t*)buf(1), (uint32_t*)buf(2), (uint32_t*)buf(3), var(0));
	} else if (p == "layer_norm_rows") {
		status = tfhip_layer_norm_rows_f32((const float*)buf(3), (const float*)buf(4), (const float*)buf(5), (float*)buf(0), (float*)buf(1), (float*)buf(2), var(0), var(1), real(2));
	} else if (p == "layer_norm_rows_backward") {
		status = tfhip_layer_norm_rows_backward_f32((const float*)buf(3), (const float*)buf(4), (const float*)buf(5), (const float*)buf(6), (const float*)buf(7), (float*)buf(0), (float*)buf(1),
		                                            (float*)buf(2), var(0), var(1));
	} else if (p == "embedding_rows") {
		status = tfhip_embedding_rows_f32((const int32_t*)buf(1), (const float*)buf(2), (float*)buf(0), var(0), var(1), var(2), real(3));
	} else if (p == "embedding_rows_backward") {
		status = tfhip_embedding_rows_backward_f32((const int32_t*)buf(1), (const float*)buf(2), (float*)buf(0), var(0), var(1), var(2), real(3));
	} else if (p == "newton_schulz") {
		const int steps = (int)var(3);
		std::vector<float> coefficients;
		for (int k = 0; k < steps && k < 64; k++)
			for (size_t i = 0; i < 3; i++) coefficients.push_back(real(5 + i));
		status = tfhip_newton_schulz_f32((const float*)buf(1), (float*)buf(0), var(0), var(1), var(2), steps, coefficients.data(), real(4));
	} else {
		throw std::runtime_error("Unknown primitive " + p);
	}
	Check(status, "Primitive " + p + " failed");
}

// A kernel recognised as one lowered reduction / prefix-sum / matmul loop: evaluates its extents and strides
// for this dispatch and runs the primitive when the operands are dense. Returns false to fall back to the
// emitted kernel (which computes the same thing for any strides).
static bool TryDispatchIdiom(const HipKernelInfo* kernel, const TFDispatchInfo& info, HipKernelManager* manager) {
	const IdiomMatchInfo& m = kernel->match;
	if (m.kind != IdiomMatchInfo::Reduce && m.kind != IdiomMatchInfo::Scan && m.kind != IdiomMatchInfo::Matmul) return false;  // the others are served only as chains
	if (!manager->idioms_enabled) return false;
	const size_t n_tensors = info.read_write_count + info.read_only_count;
	if (n_tensors != kernel->tensor_count) return false;
	if (info.variable_count != kernel->variable_count + 1 || info.variables[info.variable_count - 1] != 0) return false;
	auto buf = [&](int i) -> uint32_t* {
		const TFTensor& t = (size_t)i < info.read_write_count ? info.read_write_tensors[i] : info.read_only_tensors[i - info.read_write_count];
		return (uint32_t*)((TFHipBuffer*)t.buffer)->GetNative();
	};
	for (auto& c : m.conditions)
		if (c.first.Eval(info.variables) > c.second.Eval(info.variables)) return false;
	std::vector<long> d;
	for (const DimExpr& e : m.dims) d.push_back(e.Eval(info.variables));
	for (size_t i = 0; i < d.size(); i++)
		if (d[i] < (i < 2 ? 1 : 0)) return false;  // extents at least 1, strides never negative
	int status;
	if (m.kind == IdiomMatchInfo::Reduce) {
		long T = d[0];
		const long K = d[1], in_t = d[2], in_k = d[3], out_t = d[4];
		const int code = m.op == "sum" ? TFHIP_REDUCE_SUM : m.op == "max" ? TFHIP_REDUCE_MAX : TFHIP_REDUCE_MIN;
		if (d.size() == 8) {
			// 2-D kernel (a reduction OptimizeReductions has split into chunks): outer index with extent T1
			const long T1 = d[5], in_t1 = d[6], out_t1 = d[7];
			if (T1 < 1) return false;
			if (in_k == 1 && in_t == K && in_t1 == T * K && out_t == 1 && out_t1 == T) {
				T *= T1;  // chunks of one row follow each other: [T1 * T] rows of K
			} else if (in_t == 1 && in_k == T && in_t1 == K * T && out_t == 1 && out_t1 == T) {
				// chunks of K rows under each other: one launch of the slab-wise column reduction
				Check(tfhip_reduce_cols_slabs_f32(code, (const float*)buf(m.buffers[1]), (float*)buf(m.buffers[0]), (size_t)(T1 * K), (size_t)T, (size_t)K),
				      "Primitive for kernel " + std::to_string(info.kernel_id) + " failed");
				return true;
			} else {
				return false;
			}
		}
		if (out_t != 1 && T != 1) return false;
		if ((in_k == 1 || K == 1) && (in_t == K || T == 1))
			status = tfhip_reduce_rows_f32(code, (const float*)buf(m.buffers[1]), (float*)buf(m.buffers[0]), (size_t)T, (size_t)K);
		else if ((in_t == 1 || T == 1) && (in_k == T || K == 1))
			status = tfhip_reduce_cols_f32(code, (const float*)buf(m.buffers[1]), (float*)buf(m.buffers[0]), (size_t)K, (size_t)T);
		else
			return false;
	} else if (m.kind == IdiomMatchInfo::Scan) {
		const long T = d[0], K = d[1], in_t = d[2], in_k = d[3], out_t = d[4], out_k = d[5];
		const uint32_t* in = buf(m.buffers[1]);
		uint32_t* out = buf(m.buffers[0]);
		const bool is_float = m.is_float;
		long batch = 1, in_b = 0, out_b = 0;  // outer thread index of a 2-D kernel
		if (d.size() == 9) {
			batch = d[6];
			in_b = d[7];
			out_b = d[8];
			if (batch < 1) return false;
		}
		const bool same = in_t == out_t && in_k == out_k && in_b == out_b;
		if (same && in_k == 1 && (T == 1 || in_t == K) && (batch == 1 || in_b == T * K)) {
			// lines that follow each other in memory, each scanned along its own contiguous axis
			status = is_float ? tfhip_scan_inclusive_rows_f32((const float*)in, (float*)out, (size_t)(T * batch), (size_t)K)
			                  : tfhip_scan_inclusive_rows_u32(in, out, (size_t)(T * batch), (size_t)K);
		} else if (same && in_t == 1 && in_k == T && (batch == 1 || in_b == T * K)) {
			// down the columns of [K, T] matrices that follow each other
			status = is_float ? tfhip_scan_inclusive_cols_f32((const float*)in, (float*)out, (size_t)batch, (size_t)K, (size_t)T)
			                  : tfhip_scan_inclusive_cols_u32(in, out, (size_t)batch, (size_t)K, (size_t)T);
		} else {
			return false;
		}
	} else {
		if (m.op == "tail") {
			const long N = d[0], M = d[1], K = d[2], a_i = d[3], a_k = d[4], b_k = d[5], b_j = d[6];
			if (K < 1 || !kernel->has_tail_kernel) return false;
			const bool a_plain = (a_k == 1 || K == 1) && (a_i == K || M == 1);
			const bool a_transposed = (a_i == 1 || M == 1) && (a_k == M || K == 1);
			const bool b_plain = (b_j == 1 || N == 1) && (b_k == N || K == 1);
			const bool b_transposed = (b_k == 1 || K == 1) && (b_j == K || N == 1);
			const int layout = a_plain && b_plain ? TFHIP_GEMM_NN : a_plain && b_transposed ? TFHIP_GEMM_NT : a_transposed && b_plain ? TFHIP_GEMM_TN : -1;
			if (layout < 0) return false;
			// product[M, N] in a pooled temporary; the stream's order lets the pool hand it on right after the launch
			TFTensor* product = global_memory_manager->AllocateTensor({(size_t)M, (size_t)N}, TFSHIM_FLOAT32, "matmul_product");
			try {
				Check(tfhip_sgemm_fused(layout, (const float*)buf(m.buffers[1]), (const float*)buf(m.buffers[2]), (float*)((TFHipBuffer*)product->buffer)->GetNative(),
				                        (size_t)M, (size_t)N, (size_t)K, TFHIP_EPILOGUE_NONE, nullptr),
				      "Primitive for kernel " + std::to_string(info.kernel_id) + " failed");
				std::vector<TFTensor> tensors;
				for (size_t i = 0; i < info.read_write_count; i++) tensors.push_back(info.read_write_tensors[i]);
				for (size_t i = 0; i < info.read_only_count; i++) tensors.push_back(info.read_only_tensors[i]);
				tensors.push_back(*product);
				TFDispatchInfo tail = info;
				tail.kernel_id = kernel->tail_kernel_id;
				tail.read_write_count = tensors.size();
				tail.read_write_tensors = tensors.data();
				tail.read_only_count = 0;
				tail.read_only_tensors = nullptr;
				manager->DispatchNow(tail);
				manager->FlushBatch();  // the tail reads the temporary, which returns to the pool below
				manager->dispatch_count--;  // the pair counts as the one dispatch the host issued
			} catch (...) {
				global_memory_manager->DeallocateTensor(*product);
				throw;
			}
			global_memory_manager->DeallocateTensor(*product);
			return true;
		}
		const long N = d[0], M = d[1], K = d[2], a_i = d[3], a_k = d[4], b_k = d[5], b_j = d[6], c_i = d[7], c_j = d[8];
		if (K < 1 || (c_j != 1 && N != 1) || (c_i != N && M != 1)) return false;
		const bool a_plain = (a_k == 1 || K == 1) && (a_i == K || M == 1);
		const bool a_transposed = (a_i == 1 || M == 1) && (a_k == M || K == 1);
		const bool b_plain = (b_j == 1 || N == 1) && (b_k == N || K == 1);
		const bool b_transposed = (b_k == 1 || K == 1) && (b_j == K || N == 1);
		const float* A = (const float*)buf(m.buffers[1]);
		const float* B = (const float*)buf(m.buffers[2]);
		float* C = (float*)buf(m.buffers[0]);
		const int epilogue = m.op.empty() ? TFHIP_EPILOGUE_NONE : m.op == "bias" ? TFHIP_EPILOGUE_BIAS : m.op == "bias_relu" ? TFHIP_EPILOGUE_BIAS_RELU : TFHIP_EPILOGUE_MASK_POSITIVE;
		const float* aux = epilogue ? (const float*)buf(m.buffers[3]) : nullptr;
		const int layout = a_plain && b_plain ? TFHIP_GEMM_NN : a_plain && b_transposed ? TFHIP_GEMM_NT : a_transposed && b_plain ? TFHIP_GEMM_TN : -1;
		if (layout < 0) return false;
		if (d.size() == 13) {
			// batched: d[9] products, matrix t of A / B / C starts d[10] / d[11] / d[12] words after matrix t - 1
			const long T = d[9], a_t = d[10], b_t = d[11], c_t = d[12];
			if (T < 1 || T > 65535 || c_t < M * N || (a_t != 0 && a_t < M * K) || (b_t != 0 && b_t < K * N)) return false;
			status = tfhip_sgemm_batched(layout, A, B, C, (size_t)M, (size_t)N, (size_t)K, (size_t)T, (size_t)a_t, (size_t)b_t, (size_t)c_t);
		} else {
			status = tfhip_sgemm_fused(layout, A, B, C, (size_t)M, (size_t)N, (size_t)K, epilogue, aux);
		}
	}
	Check(status, "Primitive for kernel " + std::to_string(info.kernel_id) + " failed");
	return true;
}

// ---- chains of dispatches ---------------------------------------------------------------------------------------

void HipKernelManager::RefreshOptions() {
	idioms_enabled = std::getenv("TFHIP_NO_IDIOMS") == nullptr;
	trace_chains = std::getenv("TFHIP_TRACE_CHAINS") != nullptr;
	gather_enabled = std::getenv("TFHIP_NO_GATHER") == nullptr;
}

void HipKernelManager::Hold(const TFDispatchInfo& info) { HoldInto(chain.dispatches, info); }

// A chain has just been served: nothing of it stays behind (a stale operand would make the next chain look
// incomplete), and the buffers released while it was held return to the pool.
void HipKernelManager::FinishChain() {
	std::vector<TFTensor> frees = std::move(chain.frees);
	chain = DispatchChain();
	chain.frees = std::move(frees);
	FlushChain();
}

void HipKernelManager::HoldInto(std::vector<Deferred>& list, const TFDispatchInfo& info) {
	list.emplace_back();
	Deferred& d = list.back();
	d.tensors.assign(info.read_write_tensors, info.read_write_tensors + info.read_write_count);
	d.tensors.insert(d.tensors.end(), info.read_only_tensors, info.read_only_tensors + info.read_only_count);
	d.variables.assign(info.variables, info.variables + info.variable_count);
	d.info = info;  // the pointers are set when it runs: the vectors may still move
}

// A split reduction whose two stages are held and whose chunk tensor the program has released: one call of the
// reduction primitive on the original matrix. Returns false when that is not the state of the chain.
bool HipKernelManager::RunSplitReductionWhole() {
	if (chain.dispatches.size() != 2 || !chain.chunk_max || !chain.row_max || chain.chunk_sum || chain.row_sum) return false;
	bool released = false;
	for (const TFTensor& t : chain.frees) released |= t.buffer == chain.chunk_max;
	if (!released) return false;
	FlushBatch();
	auto ptr = [](TFBuffer* b) { return (float*)((TFHipBuffer*)b)->GetNative(); };
	const int code = chain.op == "sum" ? TFHIP_REDUCE_SUM : chain.op == "max" ? TFHIP_REDUCE_MAX : TFHIP_REDUCE_MIN;
	Check((chain.down ? tfhip_reduce_cols_f32 : tfhip_reduce_rows_f32)(code, ptr(chain.x), ptr(chain.row_max), (size_t)chain.rows, (size_t)chain.cols),
	      "Primitive for the kernels up to " + std::to_string(chain.dispatches.back().info.kernel_id) + " failed");
	dispatch_count += 2;
	idiom_dispatch_count += 2;
	fused_chain_count++;
	chain.dispatches.clear();
	return true;
}

// Row maxima and row sums of exp(x - max) are both held (two to four dispatches) and the next thing is not the
// normalising kernel: a log-softmax, a cross-entropy, ... One call computes both statistics from one read of x.
bool HipKernelManager::RunSoftmaxStatistics() {
	if (chain.stage != 4 || !chain.row_max || !chain.row_sum) return false;
	for (TFBuffer* chunk : {chain.chunk_max, chain.chunk_sum}) {
		if (!chunk) continue;
		bool released = false;
		for (const TFTensor& t : chain.frees) released |= t.buffer == chunk;
		if (!released) return false;
	}
	FlushBatch();
	auto ptr = [](TFBuffer* b) { return (float*)((TFHipBuffer*)b)->GetNative(); };
	Check(tfhip_softmax_rows_stats_f32(ptr(chain.x), nullptr, ptr(chain.row_max), ptr(chain.row_sum), (size_t)chain.rows, (size_t)chain.cols),
	      "Primitive for the kernels up to " + std::to_string(chain.dispatches.back().info.kernel_id) + " failed");
	dispatch_count += chain.dispatches.size();
	idiom_dispatch_count += chain.dispatches.size();
	fused_chain_count++;
	chain.dispatches.clear();
	return true;
}

// The softmax with e = exp(x - max) as a tensor of its own, all of it held (max, E, sums over E, Y = E / sums) and E,
// like the chunk tensors, released by the program: nobody can read E, so the fused kernel writes Y and the two row
// statistics from one read of x and E is never written.
bool HipKernelManager::RunSeparateExpSoftmax() {
	if (chain.stage != 10 || !chain.e || !chain.y || !chain.row_max || !chain.row_sum) return false;
	for (TFBuffer* skipped : {chain.e, chain.chunk_max, chain.chunk_sum}) {
		if (!skipped) continue;
		bool released = false;
		for (const TFTensor& t : chain.frees) released |= t.buffer == skipped;
		if (!released) return false;
	}
	FlushBatch();
	auto ptr = [](TFBuffer* b) { return (float*)((TFHipBuffer*)b)->GetNative(); };
	Check(tfhip_softmax_rows_stats_f32(ptr(chain.x), ptr(chain.y), ptr(chain.row_max), ptr(chain.row_sum), (size_t)chain.rows, (size_t)chain.cols),
	      "Primitive for the kernels up to " + std::to_string(chain.dispatches.back().info.kernel_id) + " failed");
	dispatch_count += chain.dispatches.size();
	idiom_dispatch_count += chain.dispatches.size();
	fused_chain_count++;
	chain.dispatches.clear();
	return true;
}

void HipKernelManager::DeferFree(TFTensor tensor) {
	if (sort.state != SortRegion::Idle) {
		sort.frees.push_back(tensor);
		if (sort.state == SortRegion::Closed && SortRegionReleased()) RunSortRegion();
		return;
	}
	if (chain.stage == 0 && batch.calls != 0) {
		batch.frees.push_back(tensor);  // nothing else is held: the buffer returns to the pool when the gathered dispatches have left
		return;
	}
	chain.frees.push_back(tensor);
	// a complete split reduction only waited to learn that nobody reads its chunk results
	if (chain.stage == 5 && tensor.buffer == chain.chunk_max) FlushChain();
	// likewise the softmax whose exponentials were a tensor of their own
	if (chain.stage == 10 && tensor.buffer == chain.e) FlushChain();
}

void HipKernelManager::RunHeld(std::vector<Deferred>& dispatches, std::vector<TFTensor>& frees, std::exception_ptr error) {
	for (Deferred& d : dispatches) {
		if (error) break;
		TFDispatchInfo info = d.info;
		info.read_write_tensors = d.tensors.data();
		info.read_only_tensors = d.tensors.data() + info.read_write_count;
		info.variables = d.variables.data();
		try {
			DispatchNow(info);
		} catch (...) {
			error = std::current_exception();
		}
	}
	if (!frees.empty()) {
		try {
			FlushBatch();  // a gathered dispatch may still name one of these buffers
		} catch (...) {
			if (!error) error = std::current_exception();
		}
	}
	for (TFTensor& t : frees) global_memory_manager->DeallocateTensor(t);
	if (error) std::rethrow_exception(error);
}

bool HipKernelManager::Batchable(const HipKernelInfo* kernel, const TFDispatchInfo& info) const {
	if (!gather_enabled) return false;
	if (kernel == nullptr || !kernel->primitive.empty() || kernel->batch_entry.empty() || kernel->has_dense_variant ||
	    (kernel->match.kind != IdiomMatchInfo::None && kernel->match.kind != IdiomMatchInfo::ExpDiff && kernel->match.kind != IdiomMatchInfo::DivideRows))
		return false;
	if (batch_handles.find(kernel->kernel_id) == batch_handles.end()) return false;
	if (info.read_write_count + info.read_only_count != kernel->tensor_count || info.variable_count != kernel->variable_count + 1) return false;  // DispatchNow reports it
	uint64_t logical = info.work_group_count;
	for (int g : kernel->group_size) logical *= (uint64_t)g;
	// the dispatches that take the one-thread-per-lane entry point: fewer threads than fill the chip
	if (kernel->idiom == "flat:vec4") return !kernel->scalar_entry.empty() && logical < (uint64_t)compute_units * (kernel->serial_load_loops ? 4096 : 1024);
	return kernel->idiom == "flat" && logical < (uint64_t)compute_units * 1024;
}

// Hazards between gathered dispatches are decided by byte ranges (device address + the buffer's extent), so buffers that
// share an allocation are told apart correctly, and by which bindings the kernel writes: the first read_write_count
// tensors of a dispatch, which is the order the generated host program passes them in (written ones first,
// Backend/CodeGen/Langs/CPP.cpp:485-491). A host that passed written tensors anywhere else would have to say so in
// HipKernelInfo::read_write_count.
void HipKernelManager::Gather(const HipKernelInfo* kernel, void* const* buffers, const size_t* buffer_bytes, size_t n_buffers, const uint32_t* vars, size_t n_vars, uint32_t grid,
                              uint32_t threads) {
	const size_t call_bytes = (size_t)kernel->batch_call_bytes;
	if (n_buffers * 8 + n_vars * 4 + 4 > call_bytes) throw std::runtime_error("Arguments of kernel " + std::to_string(kernel->kernel_id) + " do not fit its gathered form");
	bool fits = batch.calls != 0 && batch.kernel_id == kernel->kernel_id && batch.calls < (unsigned)kernel->batch_capacity && batch.threads == threads;
	for (size_t i = 0; fits && i < n_buffers; i++) {
		const bool written = i < kernel->read_write_count;
		const char* lo = (const char*)buffers[i];
		const char* hi = lo + buffer_bytes[i];
		for (auto& b : batch.buffers)
			if (lo < b.end && b.begin < hi && (b.written || written)) fits = false;
	}
	if (!fits) {
		// what is gathered leaves; buffers released since stay out of the pool until this dispatch has left too
		std::vector<TFTensor> frees = std::move(batch.frees);
		batch.frees.clear();
		FlushBatch();
		batch.frees = std::move(frees);
	}
	if (batch.calls == 0) {
		batch.kernel_id = kernel->kernel_id;
		batch.kernel = kernel;
		batch.threads = threads;
		batch.grid = 0;
		batch.arguments.assign(call_bytes * (size_t)kernel->batch_capacity, 0);
		batch.buffers.clear();
	}
	unsigned char* call = batch.arguments.data() + call_bytes * batch.calls;
	for (size_t i = 0; i < n_buffers; i++) {
		memcpy(call + 8 * i, &buffers[i], 8);
		batch.buffers.push_back({(const char*)buffers[i], (const char*)buffers[i] + buffer_bytes[i], i < kernel->read_write_count});
	}
	memcpy(call + 8 * n_buffers, vars, 4 * n_vars);
	memcpy(call + 8 * n_buffers + 4 * n_vars, &grid, 4);
	if (grid > batch.grid) batch.grid = grid;
	batch.calls++;
}

void HipKernelManager::FlushBatch() {
	if (batch.calls == 0 && batch.frees.empty()) return;
	Batch b = std::move(batch);
	batch = Batch();
	std::exception_ptr error;
	if (b.calls != 0) {
		try {
			Check(tfhip_launch_batch(batch_handles.at(b.kernel_id), b.grid, b.calls, b.threads, b.arguments.data(), b.arguments.size()),
			      "Failed to dispatch kernel " + std::to_string(b.kernel_id));
			if (b.calls > 1) {
				batched_launch_count++;
				batched_dispatch_count += b.calls;
			}
		} catch (...) {
			error = std::current_exception();
		}
	}
	for (TFTensor& t : b.frees) global_memory_manager->DeallocateTensor(t);
	if (error) std::rethrow_exception(error);
}

void HipKernelManager::FlushDeferred() {
	FlushChain();
	FlushBatch();
}

void HipKernelManager::FlushChain() {
	if (sort.state == SortRegion::Closed && SortRegionReleased())
		RunSortRegion();
	else if (sort.state != SortRegion::Idle)
		AbandonSortRegion();
	if (chain.stage == 0 && chain.frees.empty()) return;
	if (trace_chains) fprintf(stderr, "[tfhip chains] flush at stage %d: %zu dispatches, %zu frees held\n", chain.stage, chain.dispatches.size(), chain.frees.size());
	DispatchChain held;
	std::exception_ptr error;
	try {
		if (chain.stage == 5 || chain.stage == 2) RunSplitReductionWhole();
		if (chain.stage == 4) RunSoftmaxStatistics();
		if (chain.stage == 10) RunSeparateExpSoftmax();
	} catch (...) {
		error = std::current_exception();
		chain.dispatches.clear();
	}
	held = std::move(chain);
	chain = DispatchChain();
	RunHeld(held.dispatches, held.frees, error);
}

namespace {

TFBuffer* BufferAt(const TFDispatchInfo& info, int i) {
	return ((size_t)i < info.read_write_count ? info.read_write_tensors[i] : info.read_only_tensors[i - info.read_write_count]).buffer;
}

// The extents and strides of a recognised kernel for this dispatch; false when the dispatch is not what the match was made for.
bool EvaluateMatch(const HipKernelInfo* kernel, const TFDispatchInfo& info, std::vector<long>& d) {
	const IdiomMatchInfo& m = kernel->match;
	if (info.read_write_count + info.read_only_count != kernel->tensor_count) return false;
	if (info.variable_count != kernel->variable_count + 1 || info.variables[info.variable_count - 1] != 0) return false;
	for (auto& c : m.conditions)
		if (c.first.Eval(info.variables) > c.second.Eval(info.variables)) return false;
	for (const DimExpr& e : m.dims) d.push_back(e.Eval(info.variables));
	return true;
}

}  // namespace

// A plain product C[M,N] = A[K,M]^T B[K,N] on dense operands, named as a primitive or recognised from its loop.
bool HipKernelManager::HoldWeightGradient(const HipKernelInfo* kernel, const TFDispatchInfo& info) {
	if (!idioms_enabled || chain.stage != 0) return false;
	long M, N, K;
	TFBuffer *a, *b, *c;
	if (kernel->primitive == "sgemm_tn") {
		if (info.read_write_count + info.read_only_count != 3 || info.variable_count != 4) return false;
		c = BufferAt(info, 0), a = BufferAt(info, 1), b = BufferAt(info, 2);
		M = info.variables[0], N = info.variables[1], K = info.variables[2];
	} else if (kernel->primitive.empty() && kernel->match.kind == IdiomMatchInfo::Matmul && kernel->match.op.empty()) {
		std::vector<long> d;
		if (!EvaluateMatch(kernel, info, d) || d.size() != 9) return false;
		N = d[0], M = d[1], K = d[2];
		const long a_i = d[3], a_k = d[4], b_k = d[5], b_j = d[6], c_i = d[7], c_j = d[8];
		if (K < 2 || M < 2 || N < 2 || c_j != 1 || c_i != N) return false;
		if (!(a_i == 1 && a_k == M && b_j == 1 && b_k == N)) return false;  // A walked down its columns, B along its rows: tn
		c = BufferAt(info, kernel->match.buffers[0]), a = BufferAt(info, kernel->match.buffers[1]), b = BufferAt(info, kernel->match.buffers[2]);
	} else {
		return false;
	}
	if (M < 1 || N < 1 || K < 1 || a == c || b == c) return false;
	chain.stage = 6;
	chain.x = b;
	chain.a = a;
	chain.c = c;
	chain.m = M;
	chain.rows = K;
	chain.cols = N;
	Hold(info);
	return true;
}

// The column sums of the dY that the held product reads: both from one call. Anything else leaves the product to be flushed.
bool HipKernelManager::CompleteGradientPair(const HipKernelInfo* kernel, const TFDispatchInfo& info) {
	if (chain.stage != 6) return false;
	TFBuffer *in, *out;
	long rows, cols;
	if (kernel->primitive == "reduce_cols_sum") {
		if (info.read_write_count + info.read_only_count != 2 || info.variable_count != 3) return false;
		out = BufferAt(info, 0), in = BufferAt(info, 1);
		rows = info.variables[0], cols = info.variables[1];
	} else if (kernel->primitive.empty() && kernel->match.kind == IdiomMatchInfo::Reduce && kernel->match.op == "sum" && kernel->match.is_float) {
		std::vector<long> d;
		if (!EvaluateMatch(kernel, info, d) || d.size() != 5) return false;
		const long T = d[0], K = d[1], in_t = d[2], in_k = d[3], out_t = d[4];
		if (!(in_t == 1 && in_k == T && out_t == 1)) return false;  // a thread per column, walking down the rows
		rows = K, cols = T;
		out = BufferAt(info, kernel->match.buffers[0]), in = BufferAt(info, kernel->match.buffers[1]);
	} else {
		return false;
	}
	if (in != chain.x || rows != chain.rows || cols != chain.cols || out == chain.x || out == chain.a || out == chain.c) return false;
	auto ptr = [](TFBuffer* b) { return (float*)((TFHipBuffer*)b)->GetNative(); };
	FlushBatch();
	Check(tfhip_sgemm_tn_colsum(ptr(chain.a), ptr(chain.x), ptr(chain.c), ptr(out), (size_t)chain.m, (size_t)chain.cols, (size_t)chain.rows),
	      "Primitive for the kernels up to " + std::to_string(info.kernel_id) + " failed");
	dispatch_count += 2;
	idiom_dispatch_count += 2;
	fused_chain_count++;
	FinishChain();
	return true;
}

// The bias gradient was dispatched first and is held (stage 11); this is the product X^T dY over the same dY.
bool HipKernelManager::CompleteGradientPairReversed(const HipKernelInfo* kernel, const TFDispatchInfo& info) {
	if (chain.stage != 11) return false;
	long M, N, K;
	TFBuffer *a, *b, *c;
	if (kernel->primitive == "sgemm_tn") {
		if (info.read_write_count + info.read_only_count != 3 || info.variable_count != 4) return false;
		c = BufferAt(info, 0), a = BufferAt(info, 1), b = BufferAt(info, 2);
		M = info.variables[0], N = info.variables[1], K = info.variables[2];
	} else if (kernel->primitive.empty() && kernel->match.kind == IdiomMatchInfo::Matmul && kernel->match.op.empty()) {
		std::vector<long> d;
		if (!EvaluateMatch(kernel, info, d) || d.size() != 9) return false;
		N = d[0], M = d[1], K = d[2];
		const long a_i = d[3], a_k = d[4], b_k = d[5], b_j = d[6], c_i = d[7], c_j = d[8];
		if (K < 2 || M < 2 || N < 2 || c_j != 1 || c_i != N) return false;
		if (!(a_i == 1 && a_k == M && b_j == 1 && b_k == N)) return false;
		c = BufferAt(info, kernel->match.buffers[0]), a = BufferAt(info, kernel->match.buffers[1]), b = BufferAt(info, kernel->match.buffers[2]);
	} else {
		return false;
	}
	TFBuffer* sums = chain.row_sum;
	if (b != chain.x || K != chain.rows || N != chain.cols || M < 1 || a == c || b == c || c == sums || a == sums) return false;
	auto ptr = [](TFBuffer* t) { return (float*)((TFHipBuffer*)t)->GetNative(); };
	FlushBatch();
	Check(tfhip_sgemm_tn_colsum(ptr(a), ptr(b), ptr(c), ptr(sums), (size_t)M, (size_t)N, (size_t)K), "Primitive for the kernels up to " + std::to_string(info.kernel_id) + " failed");
	dispatch_count += 2;
	idiom_dispatch_count += 2;
	fused_chain_count++;
	FinishChain();
	return true;
}

// True when the dispatch opened or continued the chain (it is then held back, or the whole chain has just run).
bool HipKernelManager::AdvanceChain(const HipKernelInfo* kernel, const TFDispatchInfo& info) {
	const IdiomMatchInfo& m = kernel->match;
	if (m.kind != IdiomMatchInfo::Reduce && m.kind != IdiomMatchInfo::ExpSum && m.kind != IdiomMatchInfo::Normalise && m.kind != IdiomMatchInfo::ExpDiff &&
	    m.kind != IdiomMatchInfo::DivideRows)
		return false;
	if (!m.is_float || !idioms_enabled) return false;
	const size_t n_tensors = info.read_write_count + info.read_only_count;
	if (n_tensors != kernel->tensor_count) return false;
	if (info.variable_count != kernel->variable_count + 1 || info.variables[info.variable_count - 1] != 0) return false;
	for (auto& c : m.conditions)
		if (c.first.Eval(info.variables) > c.second.Eval(info.variables)) return false;
	std::vector<long> d;
	for (const DimExpr& e : m.dims) d.push_back(e.Eval(info.variables));
	auto buffer = [&](int i) -> TFBuffer* {
		return ((size_t)i < info.read_write_count ? info.read_write_tensors[i] : info.read_only_tensors[i - info.read_write_count]).buffer;
	};
	// A reduction-shaped kernel (Reduce, ExpSum) over a dense matrix, along the rows: whole rows ([rows] threads, `cols`
	// steps) or, split, chunks ([rows, chunks] threads, `chunk` steps, chunks * chunk == cols; chunks == 0 for whole
	// rows). Or down the columns (`down`): whole columns ([cols] threads, `rows` steps) or slabs ([slabs, cols] threads,
	// `slab` steps, slabs * slab == rows; the slab count is then in `chunks`).
	long rows = 0, cols = 0, chunks = 0;
	bool down = false;
	const bool reduction_shaped = m.kind == IdiomMatchInfo::Reduce || m.kind == IdiomMatchInfo::ExpSum;
	const bool outer = reduction_shaped && (d.size() == 8 || d.size() == 11);
	if (reduction_shaped) {
		const long T = d[0], K = d[1], in_t = d[2], in_k = d[3], out_t = d[4];
		if (T < 1 || K < 1) return false;
		if (outer) {
			const long T1 = d[5], in_t1 = d[6], out_t1 = d[7];
			if (T1 < 1 || out_t != 1 || out_t1 != T) return false;
			if (in_k == 1 && in_t == K && in_t1 == T * K) {
				rows = T1, cols = T * K, chunks = T;
			} else if (m.kind == IdiomMatchInfo::Reduce && in_t == 1 && in_k == T && in_t1 == K * T) {
				down = true, rows = T1 * K, cols = T, chunks = T1;
			} else {
				return false;
			}
		} else if (in_k == 1 && in_t == K && out_t == 1) {
			rows = T, cols = K;
		} else if (m.kind == IdiomMatchInfo::Reduce && in_t == 1 && in_k == T && out_t == 1 && ((chain.stage == 1 && chain.down) || (chain.stage == 0 && m.op == "sum"))) {
			down = true, rows = K, cols = T;  // the second stage of a split reduction down the columns, or whole column sums (a bias gradient)
		} else {
			return false;
		}
	}
	TFBuffer* out = buffer(m.buffers[0]);
	TFBuffer* in = buffer(m.buffers[1]);
	if (trace_chains)
		fprintf(stderr, "[tfhip chains] stage %d: kernel %zu kind %d op '%s' rows %ld cols %ld chunks %ld down %d\n", chain.stage, info.kernel_id, (int)m.kind, m.op.c_str(), rows, cols,
		        chunks, (int)down);
	switch (chain.stage) {
		case 0:
			// opens a chain: the first stage of a split reduction (any operation, either axis), or whole-row maxima
			if (m.kind != IdiomMatchInfo::Reduce || in == out) return false;
			if (!chunks && down && m.op == "sum") {
				// whole column sums: held for one dispatch in case the product X^T dY over the same dY follows
				chain.x = in;
				chain.row_sum = out;
				chain.rows = rows;
				chain.cols = cols;
				chain.stage = 11;
				Hold(info);
				return true;
			}
			if (!chunks && (down || m.op != "max")) return false;
			chain.x = in;
			chain.rows = rows;
			chain.cols = cols;
			chain.op = m.op;
			chain.down = down;
			chain.chunks = chunks;
			(chunks ? chain.chunk_max : chain.row_max) = out;
			chain.stage = chunks ? 1 : 2;
			Hold(info);
			return true;
		case 1:  // the second stage: the same operation over the chunk (slab) results
			if (m.kind != IdiomMatchInfo::Reduce || m.op != chain.op || chunks || down != chain.down || in != chain.chunk_max || out == chain.x || out == in) return false;
			if (down ? (cols != chain.cols || rows != chain.chunks) : (rows != chain.rows || cols != chain.chunks)) return false;
			chain.row_max = out;
			// row maxima may be the start of a softmax; anything else is complete and waits for the release of the chunk tensor
			chain.stage = (!down && m.op == "max") ? 2 : 5;
			Hold(info);
			return true;
		case 2: {  // sums of exp(x - max): whole rows or chunks; or E = exp(x - max) as a tensor of its own
			if (m.kind == IdiomMatchInfo::ExpDiff) {
				TFBuffer* e = out;
				if (in != chain.x || buffer(m.buffers[2]) != chain.row_max || e == chain.x || e == chain.row_max || e == chain.chunk_max) return false;
				const long C = d[0], R = d[1];
				if (C != chain.cols || R != chain.rows) return false;
				// X and E dense row-major, the maxima one word per row
				if (d[2] != 1 || d[3] != C || d[4] != 1 || d[5] != C || d[6] != 0 || d[7] != 1) return false;
				chain.e = e;
				chain.stage = 7;
				Hold(info);
				return true;
			}
			if (m.kind != IdiomMatchInfo::ExpSum || down || in != chain.x || buffer(m.buffers[2]) != chain.row_max || rows != chain.rows || cols != chain.cols) return false;
			if (out == chain.x || out == chain.row_max) return false;
			// the maximum is addressed by the row alone
			const size_t at = outer ? 8 : 5;
			if (outer ? !(d[at] == 0 && d[at + 1] == 0 && d[at + 2] == 1) : !(d[at] == 1 && d[at + 1] == 0)) return false;
			(chunks ? chain.chunk_sum : chain.row_sum) = out;
			chain.sum_chunks = chunks;
			chain.stage = chunks ? 3 : 4;
			Hold(info);
			return true;
		}
		case 3:  // row sums from the chunk sums
			if (m.kind != IdiomMatchInfo::Reduce || m.op != "sum" || chunks || down || in != chain.chunk_sum || rows != chain.rows || cols != chain.sum_chunks) return false;
			if (out == chain.x || out == chain.row_max || out == in) return false;
			chain.row_sum = out;
			chain.stage = 4;
			Hold(info);
			return true;
		case 7:  // sums over E: whole rows or chunks
			if (m.kind != IdiomMatchInfo::Reduce || m.op != "sum" || down || in != chain.e || rows != chain.rows || cols != chain.cols) return false;
			if (out == chain.x || out == chain.row_max || out == chain.e) return false;
			(chunks ? chain.chunk_sum : chain.row_sum) = out;
			chain.sum_chunks = chunks;
			chain.stage = chunks ? 8 : 9;
			Hold(info);
			return true;
		case 8:  // row sums from the chunk sums of E
			if (m.kind != IdiomMatchInfo::Reduce || m.op != "sum" || chunks || down || in != chain.chunk_sum || rows != chain.rows || cols != chain.sum_chunks) return false;
			if (out == chain.x || out == chain.row_max || out == chain.e || out == in) return false;
			chain.row_sum = out;
			chain.stage = 9;
			Hold(info);
			return true;
		case 9: {  // Y = E / sums: complete, and served once the program has released E (nothing else may read it)
			if (m.kind != IdiomMatchInfo::DivideRows) return false;
			TFBuffer* y = out;
			if (in != chain.e || buffer(m.buffers[2]) != chain.row_sum) return false;
			if (y == chain.x || y == chain.row_max || y == chain.row_sum || y == chain.e || y == chain.chunk_max || y == chain.chunk_sum) return false;
			const long C = d[0], R = d[1];
			if (C != chain.cols || R != chain.rows) return false;
			if (d[2] != 1 || d[3] != C || d[4] != 1 || d[5] != C || d[6] != 0 || d[7] != 1) return false;
			chain.y = y;
			chain.stage = 10;
			Hold(info);
			return true;
		}
		case 4: {
			if (m.kind != IdiomMatchInfo::Normalise) return false;
			TFBuffer* y = out;
			if (in != chain.x || buffer(m.buffers[2]) != chain.row_max || buffer(m.buffers[3]) != chain.row_sum) return false;
			if (y == chain.x || y == chain.row_max || y == chain.row_sum) return false;
			const long C = d[0], R = d[1];
			if (C != chain.cols || R != chain.rows) return false;
			// X and Y dense row-major, maxima and sums one word per row
			if (d[2] != 1 || d[3] != C || d[4] != 1 || d[5] != C || d[6] != 0 || d[7] != 1 || d[8] != 0 || d[9] != 1) return false;
			// the chunk tensors are not written: the program must have released them already
			for (TFBuffer* chunk : {chain.chunk_max, chain.chunk_sum}) {
				if (!chunk) continue;
				bool released = false;
				for (const TFTensor& t : chain.frees) released |= t.buffer == chunk;
				if (!released || chunk == y) return false;
			}
			auto ptr = [](TFBuffer* b) { return (float*)((TFHipBuffer*)b)->GetNative(); };
			FlushBatch();
			Check((m.op == "log" ? tfhip_log_softmax_rows_stats_f32 : tfhip_softmax_rows_stats_f32)(ptr(chain.x), ptr(y), ptr(chain.row_max), ptr(chain.row_sum), (size_t)R, (size_t)C),
			      "Primitive for the kernels up to " + std::to_string(info.kernel_id) + " failed");
			const size_t served = chain.dispatches.size() + 1;
			dispatch_count += served;
			idiom_dispatch_count += served;
			fused_chain_count++;
			FinishChain();
			return true;
		}
	}
	return false;
}

void HipKernelManager::DispatchKernel(TFDispatchInfo info) {
	const HipKernelInfo* kernel = FindKernelInfo(info.kernel_id);
	if (sort.state == SortRegion::Following && FollowSortDispatch(kernel, info)) return;
	if (sort.state != SortRegion::Idle) FlushChain();  // not the composition (or the region is over): what is held runs first
	if (kernel != nullptr && chain.stage == 6 && CompleteGradientPair(kernel, info)) return;
	if (kernel != nullptr && chain.stage == 11 && CompleteGradientPairReversed(kernel, info)) return;
	if (kernel != nullptr && (chain.stage == 0 || chain.stage == 6) && (kernel->primitive == "sgemm_tn" || (kernel->primitive.empty() && kernel->match.kind == IdiomMatchInfo::Matmul))) {
		FlushChain();  // a product held before this one runs first
		if (HoldWeightGradient(kernel, info)) return;
	}
	if (kernel != nullptr && kernel->primitive.empty() && kernel->match.kind != IdiomMatchInfo::None) {
		if (AdvanceChain(kernel, info)) return;
		if (HasDeferredWork()) {
			// not the chain's next kernel: what is held back runs first; this dispatch may then open a chain of its own
			FlushChain();
			if (AdvanceChain(kernel, info)) return;
		}
	} else {
		FlushChain();
	}
	DispatchNow(info);
}

void HipKernelManager::DispatchNow(TFDispatchInfo info) {
	const HipKernelInfo* kernel = FindKernelInfo(info.kernel_id);
	if (compute_units == 0) Check(tfhip_device_info(nullptr, 0, &compute_units, nullptr), "Failed to query the device");
	const bool gather = Batchable(kernel, info);
	if (!gather) FlushBatch();  // this dispatch reaches the stream now: after what was gathered before it
	if (kernel != nullptr && !kernel->primitive.empty()) {
		DispatchPrimitive(kernel, info);
		dispatch_count++;
		return;
	}
	if (kernel != nullptr && TryDispatchIdiom(kernel, info, this)) {
		dispatch_count++;
		idiom_dispatch_count++;
		return;
	}
	if (kernel != nullptr && kernel->has_dense_variant) {
		// enough threads to fill every SIMD several times over: the thread-serial form of the loops
		std::vector<int> g = kernel->group_size;
		while (g.size() < 3) g.push_back(1);
		const uint64_t logical = (uint64_t)info.work_group_count * g[0] * g[1] * g[2];
		bool serial = logical >= (uint64_t)compute_units * 4096;
		if (kernel->idiom == "reduction:block") {
			// Loops down the columns, sliced among waves (and groups): worth it while the threads alone leave SIMDs short of
			// waves and the loop is long enough to slice. The 128-row first stage of a split column reduction over
			// [16384, 4096] (half a million threads, 128 steps each) is not: 42 us thread by thread, twice that sliced.
			serial = logical >= (uint64_t)compute_units * 256;
			if (kernel->slabs) serial = logical >= (uint64_t)compute_units * 1024 || kernel->slab_trips.Eval(info.variables) < 512;
		}
		if (serial) {
			TFDispatchInfo dense = info;
			dense.kernel_id = kernel->dense_variant_id;
			DispatchNow(dense);
			return;
		}
	}
	auto it = kernel_handles.find(info.kernel_id);
	if (it == kernel_handles.end() || kernel == nullptr) throw std::runtime_error("Kernel " + std::to_string(info.kernel_id) + " was not compiled");
	if (info.read_write_count == 0) throw std::runtime_error("No tensors provided to kernel");

	// Generated hosts pass every tensor in read_write_tensors (rw first, then ro) and none in
	// read_only_tensors (CPP.cpp:485-491); accept the split form too.
	void* buffers[66];  // the tensors, and the two buffers of a dispatch that shares a loop among HIP groups
	size_t n_buffers = 0;
	const size_t expected = kernel->tensor_count;
	if (info.read_write_count + info.read_only_count != expected)
		throw std::runtime_error("Kernel " + std::to_string(info.kernel_id) + " expects " + std::to_string(expected) + " tensors, got " +
		                         std::to_string(info.read_write_count + info.read_only_count));
	if (expected > 64) throw std::runtime_error("Too many tensors bound to one kernel");
	size_t buffer_bytes[66];  // extents, for the overlap test of gathered dispatches
	for (size_t i = 0; i < info.read_write_count; i++) {
		buffer_bytes[n_buffers] = info.read_write_tensors[i].buffer->size * sizeof(uint32_t);
		buffers[n_buffers++] = ((TFHipBuffer*)info.read_write_tensors[i].buffer)->GetNative();
	}
	for (size_t i = 0; i < info.read_only_count; i++) {
		buffer_bytes[n_buffers] = info.read_only_tensors[i].buffer->size * sizeof(uint32_t);
		buffers[n_buffers++] = ((TFHipBuffer*)info.read_only_tensors[i].buffer)->GetNative();
	}

	// Variable block: the host's words (user scalars + block offset) followed by the group count.
	const size_t expected_vars = kernel->variable_count + 1;
	if (info.variable_count != expected_vars)
		throw std::runtime_error("Kernel " + std::to_string(info.kernel_id) + " expects " + std::to_string(expected_vars) + " variable words, got " + std::to_string(info.variable_count));
	if (info.work_group_count > 0xFFFFFFFFull) throw std::runtime_error("work_group_count does not fit 32 bits");
	uint32_t vars[260];
	if (expected_vars + 1 > 258) throw std::runtime_error("Too many kernel variables");
	for (size_t i = 0; i < info.variable_count; i++) vars[i] = info.variables[i];
	vars[info.variable_count] = (uint32_t)info.work_group_count;
	size_t n_vars = info.variable_count + 1;
	TFTensor* slab_partials = nullptr;  // temporary of a dispatch that shares a loop among HIP groups, returned to the pool after the launch

	std::vector<int> group = kernel->group_size;
	while (group.size() < 3) group.push_back(1);
	uint64_t grid;
	uint32_t bx = (uint32_t)kernel->hip_threads, by = 1, bz = 1;
	tfhip_kernel_t handle = it->second;
	if (kernel->idiom == "group") {
		grid = info.work_group_count;
		bx = group[0];
		by = group[1];
		bz = group[2];
	} else if (kernel->idiom == "reduction:wave") {
		const uint64_t logical = (uint64_t)info.work_group_count * group[0] * group[1] * group[2];
		const uint64_t per_block = 256 / (uint64_t)kernel->lanes_per_thread * (uint64_t)kernel->threads_per_lane_group;
		grid = (logical + per_block - 1) / per_block;
	} else if (kernel->idiom == "reduction:block") {
		const uint64_t logical = (uint64_t)info.work_group_count * group[0] * group[1] * group[2];
		grid = (logical + 63) / 64;
		if (kernel->slabs) {
			// A loop down the columns of a matrix with few columns: so many HIP groups share each group of 64 threads, slab
			// by slab, that every compute unit has one group of sixteen waves (the mean over axis 0 of [16384, 16, 16, 16],
			// 64 groups of threads: 150 us with one slab, 50 us with four, 60-70 us with eight to thirty-two), as long as a
			// wave's slice of its slab stays 32 steps long. Their per-slab results meet in a pooled temporary.
			const uint64_t column_groups = grid;
			const long trips = kernel->slab_trips.Eval(info.variables);
			uint64_t slabs = 1;
			if (column_groups < (uint64_t)compute_units && column_groups <= kSlabTicketWords && trips >= 1024) {
				slabs = ((uint64_t)compute_units + column_groups - 1) / column_groups;
				slabs = std::min<uint64_t>(std::min<uint64_t>(slabs, (uint64_t)trips / 512), 64);
				slabs = std::max<uint64_t>(slabs, 1);
			}
			if (slab_tickets == nullptr) {
				Check(tfhip_malloc(&slab_tickets, kSlabTicketWords * sizeof(uint32_t)), "Failed to allocate the slab ticket counters");
				Check(tfhip_fill_u32(slab_tickets, 0, kSlabTicketWords), "Failed to clear the slab ticket counters");
			}
			void* partials = slab_tickets;  // with one slab the kernel touches neither buffer, but a launch takes no null pointer
			if (slabs > 1) {
				slab_partials = global_memory_manager->AllocateTensor({(size_t)(slabs * column_groups * 64 * (uint64_t)kernel->slab_words_per_thread)}, TFSHIM_FLOAT32, "slab_partials");
				partials = ((TFHipBuffer*)slab_partials->buffer)->GetNative();
			}
			buffers[n_buffers++] = partials;
			buffers[n_buffers++] = slab_tickets;
			vars[n_vars++] = (uint32_t)slabs;
			grid = column_groups * slabs;
		}
	} else {
		// "flat" and "flat:vec4": Q IR groups per tile; the grid is padded to a multiple of 8 because the
		// kernels deal tiles to the 8 dies in contiguous bands (surplus groups exit at once).
		const uint64_t logical = (uint64_t)info.work_group_count * group[0] * group[1] * group[2];
		auto scalar = scalar_handles.find(info.kernel_id);
		if (kernel->idiom == "flat:vec4" && scalar != scalar_handles.end() && logical < (uint64_t)compute_units * (kernel->serial_load_loops ? 4096 : 1024)) {
			// Fewer than one 256-thread group of quads per compute unit: run one logical thread per lane instead. A kernel
			// whose threads walk a loop of loads by themselves hides memory latency by the number of waves, so it stays
			// with one thread per lane until the quads alone give four waves per SIMD (the 128-row first stage of a
			// column reduction over [16384, 4096]: 47.7 -> 42 us).
			handle = scalar->second;
			bx = (uint32_t)kernel->scalar_hip_threads;
			grid = (info.work_group_count + kernel->scalar_groups_per_hip_block - 1) / kernel->scalar_groups_per_hip_block;
		} else if (gather && kernel->idiom == "flat:vec4") {
			throw std::runtime_error("Kernel " + std::to_string(info.kernel_id) + " has no one-thread-per-lane entry point");
		} else {
			grid = (info.work_group_count + kernel->groups_per_hip_block - 1) / kernel->groups_per_hip_block;
			grid *= kernel->hip_blocks_per_tile;
		}
		grid = (grid + 7) / 8 * 8;
		if (gather && grid <= 0x7FFFFFFFull) {
			Gather(kernel, buffers, buffer_bytes, n_buffers, vars, info.variable_count + 1, (uint32_t)grid, bx);
			dispatch_count++;
			return;
		}
	}
	if (grid > 0x7FFFFFFFull) throw std::runtime_error("Dispatch of kernel " + std::to_string(info.kernel_id) + " needs " + std::to_string(grid) + " groups, more than one launch can hold");
	const int launched = tfhip_launch(handle, (uint32_t)grid, bx, by, bz, buffers, n_buffers, vars, n_vars);
	if (slab_partials != nullptr) global_memory_manager->DeallocateTensor(*slab_partials);  // the stream's order keeps it until the kernel is done
	Check(launched, "Failed to dispatch kernel " + std::to_string(info.kernel_id));
	dispatch_count++;
}

void HipKernelManager::FreeKernel(size_t kernel_id) {
	auto sc = scalar_handles.find(kernel_id);
	if (sc != scalar_handles.end()) {
		tfhip_module_unload(sc->second);
		scalar_handles.erase(sc);
	}
	auto bt = batch_handles.find(kernel_id);
	if (bt != batch_handles.end()) {
		tfhip_module_unload(bt->second);
		batch_handles.erase(bt);
	}
	kernel_infos.erase(kernel_id);
	auto it = kernel_handles.find(kernel_id);
	if (it == kernel_handles.end()) return;
	tfhip_module_unload(it->second);
	kernel_handles.erase(it);
}

void HipKernelManager::FreeAllKernels() {
	if (slab_tickets != nullptr) {
		tfhip_free(slab_tickets);
		slab_tickets = nullptr;
	}
	for (auto& kv : scalar_handles) tfhip_module_unload(kv.second);
	scalar_handles.clear();
	for (auto& kv : batch_handles) tfhip_module_unload(kv.second);
	batch_handles.clear();
	for (auto& kv : kernel_handles) tfhip_module_unload(kv.second);
	kernel_handles.clear();
	kernel_infos.clear();
}

}  // namespace TFSHIM_NAMESPACE
