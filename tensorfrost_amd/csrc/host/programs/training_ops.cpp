// Programs around the operators of a training step that stand beside the dense layers' products. As in primitives.cpp, the
// host part is what the reference's generator would emit for such a program and the kernels are primitive-backed.
// Floating-point parameters are passed as the integer of their 32 bits; parameters that a program does not have are refused.
//
//   layer_norm            y, mean, rstd = f(x, weight, bias)                                  params: eps
//   layer_norm_backward   dx, dweight, dbias = f(x, dy, weight, mean, rstd)
//   embedding             out = f(tokens, table)                                              params: scale
//   embedding_backward    dtable = f(tokens, dy)                                              params: vocabulary, scale
//   newton_schulz         out = f(g), g [matrices, rows, cols]                                params: steps, eps, a, b, c
//   embed_norm_dense      one step of embedding -> layer norm -> dense layer, forward and backward:
//                         y, dtable, dweight, dbias, update = f(tokens, table, weight, bias, W, dy), update the orthogonalised
//                         gradient of W                                                       params: eps, scale
#include <cstdint>
#include <cstring>
#include <stdexcept>
#include <string>

#include "registry.h"

namespace tfhost {

static int Bits(float v) {
	int w;
	memcpy(&w, &v, sizeof(w));
	return w;
}
static int Param(const std::vector<int64_t>& params, size_t i, int otherwise) { return i < params.size() ? (int)params[i] : otherwise; }

// A program takes the same coefficients for all its steps, for one: triples of every step would be read as one triple.
static void CheckParams(const char* program, const std::vector<int64_t>& params, size_t most) {
	if (params.size() > most) throw std::runtime_error(std::string(program) + " takes at most " + std::to_string(most) + " parameters (got " + std::to_string(params.size()) + ")");
	for (size_t i = 0; i < params.size(); i++)
		if (params[i] < INT32_MIN || params[i] > (int64_t)UINT32_MAX) throw std::runtime_error(std::string(program) + ": parameter " + std::to_string(i) + " does not fit 32 bits");
}

static const float kLayerEps = 1e-5f, kNormEps = 1e-7f, kQuintic[3] = {3.4445f, -4.7750f, 2.0315f};

static void BuildLayerNorm(Program* program, const std::vector<int64_t>& params) {
	CheckParams("layer_norm", params, 1);
	Kernel* norm = program->AddPrimitive("layer_norm_rows", 6, 3);
	HostBuilder h(program);
	V x = h.Input("x", {-1, -1}, TFType_Float);
	V R = h.Shape(x)[0], C = h.Shape(x)[1];
	V weight = h.Input("weight", {C}, TFType_Float);
	V bias = h.Input("bias", {C}, TFType_Float);
	V y = h.Allocate("y", {R, C}, TFType_Float);
	V mean = h.Allocate("mean", {R}, TFType_Float);
	V rstd = h.Allocate("rstd", {R}, TFType_Float);
	h.Dispatch(norm, {y, mean, rstd}, {x, weight, bias}, {R, C, h.Const(Param(params, 0, Bits(kLayerEps)))}, {R, C});
	for (V out : {y, mean, rstd}) h.Output(out);
	h.Finish();
}

static void BuildLayerNormBackward(Program* program, const std::vector<int64_t>& params) {
	CheckParams("layer_norm_backward", params, 0);
	Kernel* back = program->AddPrimitive("layer_norm_rows_backward", 8, 2);
	HostBuilder h(program);
	V x = h.Input("x", {-1, -1}, TFType_Float);
	V R = h.Shape(x)[0], C = h.Shape(x)[1];
	V dy = h.Input("dy", {R, C}, TFType_Float);
	V weight = h.Input("weight", {C}, TFType_Float);
	V mean = h.Input("mean", {R}, TFType_Float);
	V rstd = h.Input("rstd", {R}, TFType_Float);
	V dx = h.Allocate("dx", {R, C}, TFType_Float);
	V dweight = h.Allocate("dweight", {C}, TFType_Float);
	V dbias = h.Allocate("dbias", {C}, TFType_Float);
	h.Dispatch(back, {dx, dweight, dbias}, {x, dy, weight, mean, rstd}, {R, C}, {R, C});
	for (V out : {dx, dweight, dbias}) h.Output(out);
	h.Finish();
}

static void BuildEmbedding(Program* program, const std::vector<int64_t>& params) {
	CheckParams("embedding", params, 1);
	Kernel* lookup = program->AddPrimitive("embedding_rows", 3, 4);
	HostBuilder h(program);
	V tokens = h.Input("tokens", {-1}, TFType_Int);
	V table = h.Input("table", {-1, -1}, TFType_Float);
	V n = h.Shape(tokens)[0], vocab = h.Shape(table)[0], C = h.Shape(table)[1];
	V out = h.Allocate("embedded", {n, C}, TFType_Float);
	h.Dispatch(lookup, {out}, {tokens, table}, {n, vocab, C, h.Const(Param(params, 0, Bits(1.0f)))}, {n, C});
	h.Output(out);
	h.Finish();
}

static void BuildEmbeddingBackward(Program* program, const std::vector<int64_t>& params) {
	CheckParams("embedding_backward", params, 2);
	if (params.empty() || params[0] < 1 || params[0] > 0x7FFFFFFF) throw std::runtime_error("embedding_backward needs the number of rows of the table as its first parameter");
	Kernel* back = program->AddPrimitive("embedding_rows_backward", 3, 4);
	HostBuilder h(program);
	V tokens = h.Input("tokens", {-1}, TFType_Int);
	V n = h.Shape(tokens)[0];
	V dy = h.Input("dy", {n, -1}, TFType_Float);
	V vocab = h.Const((int)params[0]), C = h.Shape(dy)[1];
	V dtable = h.Allocate("dtable", {vocab, C}, TFType_Float);
	h.Dispatch(back, {dtable}, {tokens, dy}, {n, vocab, C, h.Const(Param(params, 1, Bits(1.0f)))}, {n, C});
	h.Output(dtable);
	h.Finish();
}

static std::vector<V> NewtonSchulzVariables(HostBuilder& h, V batch, V rows, V cols, const std::vector<int64_t>& params) {
	std::vector<V> v = {batch, rows, cols, h.Const(Param(params, 0, 5)), h.Const(Param(params, 1, Bits(kNormEps)))};
	for (size_t i = 0; i < 3; i++) v.push_back(h.Const(Param(params, 2 + i, Bits(kQuintic[i]))));
	return v;
}

static void BuildNewtonSchulz(Program* program, const std::vector<int64_t>& params) {
	CheckParams("newton_schulz", params, 5);
	Kernel* schulz = program->AddPrimitive("newton_schulz", 2, 8);
	HostBuilder h(program);
	V g = h.Input("g", {-1, -1, -1}, TFType_Float);
	V B = h.Shape(g)[0], R = h.Shape(g)[1], C = h.Shape(g)[2];
	V out = h.Allocate("orthogonal", {B, R, C}, TFType_Float);
	h.Dispatch(schulz, {out}, {g}, NewtonSchulzVariables(h, B, R, C, params), {B, R, C});
	h.Output(out);
	h.Finish();
}

static void BuildEmbedNormDense(Program* program, const std::vector<int64_t>& params) {
	CheckParams("embed_norm_dense", params, 2);
	Kernel* lookup = program->AddPrimitive("embedding_rows", 3, 4);
	Kernel* norm = program->AddPrimitive("layer_norm_rows", 6, 3);
	Kernel* gemm_nn = program->AddPrimitive("sgemm_nn", 3, 3);
	Kernel* gemm_tn = program->AddPrimitive("sgemm_tn", 3, 3);
	Kernel* gemm_nt = program->AddPrimitive("sgemm_nt", 3, 3);
	Kernel* schulz = program->AddPrimitive("newton_schulz", 2, 8);
	Kernel* norm_back = program->AddPrimitive("layer_norm_rows_backward", 8, 2);
	Kernel* lookup_back = program->AddPrimitive("embedding_rows_backward", 3, 4);
	HostBuilder h(program);
	V tokens = h.Input("tokens", {-1}, TFType_Int);
	V table = h.Input("table", {-1, -1}, TFType_Float);
	V n = h.Shape(tokens)[0], vocab = h.Shape(table)[0], C = h.Shape(table)[1];
	V weight = h.Input("weight", {C}, TFType_Float);
	V bias = h.Input("bias", {C}, TFType_Float);
	V W = h.Input("W", {C, -1}, TFType_Float);
	V K = h.Shape(W)[1];
	V dy = h.Input("dy", {n, K}, TFType_Float);
	V eps = h.Const(Param(params, 0, Bits(kLayerEps))), scale = h.Const(Param(params, 1, Bits(1.0f)));
	// forward
	V embedded = h.Allocate("embedded", {n, C}, TFType_Float);
	V normed = h.Allocate("normed", {n, C}, TFType_Float);
	V mean = h.Allocate("mean", {n}, TFType_Float);
	V rstd = h.Allocate("rstd", {n}, TFType_Float);
	V y = h.Allocate("y", {n, K}, TFType_Float);
	h.Dispatch(lookup, {embedded}, {tokens, table}, {n, vocab, C, scale}, {n, C});
	h.Dispatch(norm, {normed, mean, rstd}, {embedded, weight, bias}, {n, C, eps}, {n, C});
	h.Dispatch(gemm_nn, {y}, {normed, W}, {n, K, C}, {n, K});
	// backward
	V dW = h.Allocate("dW", {C, K}, TFType_Float);
	V update = h.Allocate("update", {C, K}, TFType_Float);
	V dnormed = h.Allocate("dnormed", {n, C}, TFType_Float);
	V dembedded = h.Allocate("dembedded", {n, C}, TFType_Float);
	V dweight = h.Allocate("dweight", {C}, TFType_Float);
	V dbias = h.Allocate("dbias", {C}, TFType_Float);
	V dtable = h.Allocate("dtable", {vocab, C}, TFType_Float);
	h.Dispatch(gemm_tn, {dW}, {normed, dy}, {C, K, n}, {C, K});
	h.Dispatch(schulz, {update}, {dW}, NewtonSchulzVariables(h, h.Const(1), C, K, {}), {C, K});
	h.Dispatch(gemm_nt, {dnormed}, {dy, W}, {n, C, K}, {n, C});
	h.Dispatch(norm_back, {dembedded, dweight, dbias}, {embedded, dnormed, weight, mean, rstd}, {n, C}, {n, C});
	h.Dispatch(lookup_back, {dtable}, {tokens, dembedded}, {n, vocab, C, scale}, {n, C});
	for (V t : {embedded, normed, mean, rstd, dW, dnormed, dembedded}) h.Deallocate(t);
	for (V out : {y, dtable, dweight, dbias, update}) h.Output(out);
	h.Finish();
}

static ProgramRegistrar reg_norm("layer_norm", BuildLayerNorm);
static ProgramRegistrar reg_norm_back("layer_norm_backward", BuildLayerNormBackward);
static ProgramRegistrar reg_embedding("embedding", BuildEmbedding);
static ProgramRegistrar reg_embedding_back("embedding_backward", BuildEmbeddingBackward);
static ProgramRegistrar reg_schulz("newton_schulz", BuildNewtonSchulz);
static ProgramRegistrar reg_step("embed_norm_dense", BuildEmbedNormDense);

}  // namespace tfhost
