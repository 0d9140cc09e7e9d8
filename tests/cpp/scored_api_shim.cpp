// scored_api_shim.cpp - C entry points over the C++ API of scored attention, attention weights and eviction, for
// tests/test_gpu_scored_cxx.py: a decode step of a server that evicts, as an engine would write it.
#include <string>

#include "firefly/kernels.h"

using namespace firefly;

extern "C" {

const char* sas_last_error()
{
    static thread_local std::string e;
    e = kernels::last_error();
    return e.c_str();
}

// q [B, S, Hq, D] (dtype qd) over caches [N, 16, Hkv, D] (dtype cd; table null: contiguous [B, S, Hkv, D]); weights and prior
// [B, Hkv, T] or null.
int sas_attention(void* q, void* k, void* v, void* ks, void* vs, void* out, int* table, int* ctx, int B, int S, int Hq, int Hkv,
                  int D, int N, int max_blocks, int qd, int cd, float cap, float* slopes, int window, int* begin, int* end,
                  float* weights, float* prior, float decay, int T, void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType qt = static_cast<DType>(qd), ct = static_cast<DType>(cd);
    Tensor tq = Tensor::from_external(q, {B, S, Hq, D}, qt, Device::GPU);
    Tensor to = Tensor::from_external(out, {B, S, Hq * D}, qt, Device::GPU);
    Tensor kc = table ? Tensor::from_external(k, {N, 16, Hkv, D}, ct, Device::GPU)
                      : Tensor::from_external(k, {B, S, Hkv, D}, ct, Device::GPU);
    Tensor vc = table ? Tensor::from_external(v, {N, 16, Hkv, D}, ct, Device::GPU)
                      : Tensor::from_external(v, {B, S, Hkv, D}, ct, Device::GPU);
    Tensor tks = Tensor::from_external(ks, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor tvs = Tensor::from_external(vs, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor w = Tensor::from_external(weights, {B, Hkv, T}, DType::F32, Device::GPU);
    Tensor p = Tensor::from_external(prior, {B, Hkv, T}, DType::F32, Device::GPU);
    const kernels::ScoreRule rule{cap, slopes, window, begin, end};
    kernels::attention_scored(tq, kc, vc, to, table, Hkv, S, max_blocks, ctx, rule, ks ? &tks : nullptr, vs ? &tvs : nullptr,
                              weights ? &w : nullptr, prior ? &p : nullptr, decay, weights ? T : 0);
    return kernels::last_error().empty() ? 0 : -1;
}

int sas_weights(void* q, void* k, void* ks, int* table, int* ctx, int B, int S, int Hq, int Hkv, int D, int N, int max_blocks,
                int qd, int cd, float cap, float* slopes, int window, int* begin, int* end, float* weights, float* prior,
                float decay, int T, void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType qt = static_cast<DType>(qd), ct = static_cast<DType>(cd);
    Tensor tq = Tensor::from_external(q, {B, S, Hq, D}, qt, Device::GPU);
    Tensor kc = Tensor::from_external(k, {N, 16, Hkv, D}, ct, Device::GPU);
    Tensor tks = Tensor::from_external(ks, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor w = Tensor::from_external(weights, {B, Hkv, T}, DType::F32, Device::GPU);
    Tensor p = Tensor::from_external(prior, {B, Hkv, T}, DType::F32, Device::GPU);
    const kernels::ScoreRule rule{cap, slopes, window, begin, end};
    kernels::attention_weights(tq, kc, w, prior ? &p : nullptr, decay, table, Hkv, max_blocks, ctx, rule, ks ? &tks : nullptr, T);
    return kernels::last_error().empty() ? 0 : -1;
}

int sas_evict(float* weights, int T, void* k, void* v, void* ks, void* vs, int* table, int* ctx, int B, int Hkv, int D, int N,
              int max_blocks, int cd, int keep, int sinks, int recent, int* kept, int* kept_lens, int* dst, int dst_blocks,
              float* weights_out, void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType ct = static_cast<DType>(cd);
    Tensor kc = Tensor::from_external(k, {N, 16, Hkv, D}, ct, Device::GPU);
    Tensor vc = Tensor::from_external(v, {N, 16, Hkv, D}, ct, Device::GPU);
    Tensor tks = Tensor::from_external(ks, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor tvs = Tensor::from_external(vs, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor w = Tensor::from_external(weights, {B, Hkv, T}, DType::F32, Device::GPU);
    Tensor wo = Tensor::from_external(weights_out, {B, Hkv, T}, DType::F32, Device::GPU);
    Tensor tk = Tensor::from_external(kept, {B, Hkv, keep}, DType::I32, Device::GPU);
    Tensor tl = Tensor::from_external(kept_lens, {B}, DType::I32, Device::GPU);
    kernels::evict_kv_cache(w, kc, vc, table, ctx, max_blocks, keep, sinks, recent, tk, tl, dst, dst_blocks,
                            weights_out ? &wo : nullptr, ks ? &tks : nullptr, vs ? &tvs : nullptr);
    return kernels::last_error().empty() ? 0 : -1;
}

}  // extern "C"
