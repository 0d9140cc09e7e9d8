// scored_prompt_shim.cpp - C entry points over the C++ API of scored attention, for tests/test_gpu_scored_prompt.py: a
// prompt's chunks of any length, one token among them, and a decode step with its append, as an engine would write them.
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

// A decode step: q [B, 1, Hq, D] over caches [N, 16, Hkv, D] (dtype cd; scales [N, 16, Hkv] or null) with new tokens
// [B, S, Hkv, D] (either may be null), weights and prior [B, Hkv, T] or null.
int sps_step(void* q, void* k, void* v, void* ks, void* vs, void* out, int* table, int* ctx, int B, int S, int Hq, int Hkv, int D,
             int N, int max_blocks, int dt, int cd, int window, void* k_new, void* v_new, float* weights, float* prior, int T,
             int prefill, void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType t = static_cast<DType>(dt), c = static_cast<DType>(cd);
    Tensor tq = Tensor::from_external(q, {B, 1, Hq, D}, t, Device::GPU);
    Tensor to = Tensor::from_external(out, {B, 1, Hq * D}, t, Device::GPU);
    Tensor kc = Tensor::from_external(k, {N, 16, Hkv, D}, c, Device::GPU);
    Tensor vc = Tensor::from_external(v, {N, 16, Hkv, D}, c, Device::GPU);
    Tensor tks = Tensor::from_external(ks, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor tvs = Tensor::from_external(vs, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor kn = Tensor::from_external(k_new, {B, S, Hkv, D}, t, Device::GPU);
    Tensor vn = Tensor::from_external(v_new, {B, S, Hkv, D}, t, Device::GPU);
    Tensor w = Tensor::from_external(weights, {B, Hkv, T}, DType::F32, Device::GPU);
    Tensor p = Tensor::from_external(prior, {B, Hkv, T}, DType::F32, Device::GPU);
    kernels::ScoreRule rule{};
    rule.window = window;
    rule.prefill = prefill != 0;
    kernels::attention_scored(tq, kc, vc, to, table, Hkv, 1, max_blocks, ctx, rule, ks ? &tks : nullptr, vs ? &tvs : nullptr,
                              weights ? &w : nullptr, prior ? &p : nullptr, 0.5f, weights ? T : 0, k_new ? &kn : nullptr,
                              v_new ? &vn : nullptr);
    return kernels::last_error().empty() ? 0 : -1;
}

// Call `op` over caches of 4 pages of `block` tokens, nothing of which is read where the call is refused; rows 0: no rows.
int sps_block_size(int op, int block, int rows)
{
    void* const p = reinterpret_cast<void*>(uintptr_t{256});
    int* const  i = static_cast<int*>(p);
    const int   S = op == 1 || op == 3 ? 2 : 1;
    Tensor      q = Tensor::from_external(p, {rows, S, 4, 64}, DType::BF16, Device::GPU);
    Tensor      o = Tensor::from_external(p, {rows, S, 256}, DType::BF16, Device::GPU);
    Tensor      n = Tensor::from_external(p, {rows, 1, 2, 64}, DType::BF16, Device::GPU);
    Tensor      k = Tensor::from_external(p, {4, block, 2, 64}, DType::BF16, Device::GPU);
    Tensor      v = Tensor::from_external(p, {4, block, 2, 64}, DType::BF16, Device::GPU);
    Tensor      w = Tensor::from_external(p, {rows, 2, 64}, DType::F32, Device::GPU);
    const kernels::ScoreRule rule{};
    switch (op)
    {
        case 0:
        case 1: kernels::attention_scored(q, k, v, o, p, 2, S, 4, i, rule); break;
        case 2:
        case 3: kernels::attention(q, k, v, o, p, 2, S, 4, i); break;
        case 4: kernels::attention_weights(q, k, w, nullptr, 1.0f, i, 2, 4, i, rule); break;
        case 5: kernels::attention_shared_prefix(q, k, v, o, p, 2, 4, i, 1); break;
        default: kernels::append_kv_cache_attention(n, n, q, k, v, o, p, 2, 4, i);
    }
    return kernels::last_error().empty() ? 0 : -1;
}

}  // extern "C"
