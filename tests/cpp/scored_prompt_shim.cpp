// scored_prompt_shim.cpp - C entry points over the C++ API of scored attention, for tests/test_gpu_scored_prompt.py: a
// prompt's chunks of any length, one token among them, as an engine would write them.
#include <string>

#include "firefly/kernels.h"

using namespace firefly;

extern "C" {

const char* sps_last_error()
{
    static thread_local std::string e;
    e = kernels::last_error();
    return e.c_str();
}

// q [B, S, Hq, D] over caches [N, 16, Hkv, D], all of dtype dt; prefill: ScoreRule::prefill.
int sps_attention(void* q, void* k, void* v, void* out, int* table, int* ctx, int B, int S, int Hq, int Hkv, int D, int N,
                  int max_blocks, int dt, float cap, int window, int* begin, int* end, int prefill, void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType t = static_cast<DType>(dt);
    Tensor tq = Tensor::from_external(q, {B, S, Hq, D}, t, Device::GPU);
    Tensor to = Tensor::from_external(out, {B, S, Hq * D}, t, Device::GPU);
    Tensor kc = Tensor::from_external(k, {N, 16, Hkv, D}, t, Device::GPU);
    Tensor vc = Tensor::from_external(v, {N, 16, Hkv, D}, t, Device::GPU);
    const kernels::ScoreRule rule{cap, nullptr, window, begin, end, prefill != 0};
    kernels::attention_scored(tq, kc, vc, to, table, Hkv, S, max_blocks, ctx, rule);
    return kernels::last_error().empty() ? 0 : -1;
}

}  // extern "C"
