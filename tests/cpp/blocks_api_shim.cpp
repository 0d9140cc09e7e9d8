// blocks_api_shim.cpp - C entry points over the C++ API of rotary positions on several axes, key bounds, the choice of pages
// and the attention over them, for tests/test_gpu_blocks_cxx.py: a step or chunk as an engine would write it.
#include <string>

#include "firefly/kernels.h"

using namespace firefly;

extern "C" {

const char* bas_last_error()
{
    static thread_local std::string e;
    e = kernels::last_error();
    return e.c_str();
}

// One layer's calls: q [B, S, Hq, D] rotated and k, v [B, S, Hkv, D] appended to caches [N, 16, Hkv, D] (dtype cd, scales or
// null), the bounds [N, Hkv, 2, D] of their pages, the lists, and the attention over them.
int bas_layer(void* q, void* k, void* v, int* positions, const int* sections, int axes, int interleaved, void* kc, void* vc,
              void* ks, void* vs, void* bounds, int* blocks, void* out, int* table, int* ctx, int B, int S, int Hq, int Hkv, int D,
              int N, int max_blocks, int dt, int cd, int bd, int count, int sinks, int recent, int query_block, void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType t = static_cast<DType>(dt), c = static_cast<DType>(cd);
    Tensor tq = Tensor::from_external(q, {B, S, Hq, D}, t, Device::GPU);
    Tensor tk = Tensor::from_external(k, {B, S, Hkv, D}, t, Device::GPU);
    Tensor tv = Tensor::from_external(v, {B, S, Hkv, D}, t, Device::GPU);
    Tensor tkc = Tensor::from_external(kc, {N, 16, Hkv, D}, c, Device::GPU);
    Tensor tvc = Tensor::from_external(vc, {N, 16, Hkv, D}, c, Device::GPU);
    Tensor tks = Tensor::from_external(ks, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor tvs = Tensor::from_external(vs, {N, 16, Hkv}, DType::F32, Device::GPU);
    Tensor box = Tensor::from_external(bounds, {N, Hkv, 2, D}, static_cast<DType>(bd), Device::GPU);
    Tensor li = Tensor::from_external(blocks, {B, (S + query_block - 1) / query_block, Hkv, count}, DType::I32, Device::GPU);
    Tensor to = Tensor::from_external(out, {B, S, Hq * D}, t, Device::GPU);
    kernels::AxisPositions at{};
    at.positions = positions;
    at.axes = axes;
    for (int i = 0; i < axes && i < 4; ++i) at.sections[i] = sections[i];
    at.interleaved = interleaved != 0;
    Tensor* pks = ks ? &tks : nullptr;
    Tensor* pvs = vs ? &tvs : nullptr;
    auto bad = [] { return !kernels::last_error().empty(); };
    kernels::rope_append_kv_cache_axes(tq, tk, tv, tkc, tvc, table, ctx, max_blocks, at, pks, pvs);
    if (bad()) return -1;
    kernels::update_key_bounds(tkc, box, table, ctx, B, max_blocks, S, pks);
    if (bad()) return -2;
    kernels::select_blocks(tq, box, li, table, ctx, max_blocks, sinks, recent, query_block);
    if (bad()) return -3;
    kernels::attention_blocks(tq, tkc, tvc, to, li, table, ctx, max_blocks, query_block, pks, pvs);
    return bad() ? -4 : 0;
}

// apply_rope_axes in place.
int bas_rope(void* q, void* k, int* positions, const int* sections, int axes, int B, int S, int Hq, int Hkv, int D, int dt,
             void* stream)
{
    kernels::set_default_stream(static_cast<hipStream_t>(stream));
    const DType t = static_cast<DType>(dt);
    Tensor tq = Tensor::from_external(q, {B, S, Hq, D}, t, Device::GPU);
    Tensor tk = Tensor::from_external(k, {B, S, Hkv, D}, t, Device::GPU);
    kernels::AxisPositions at{};
    at.positions = positions;
    at.axes = axes;
    for (int i = 0; i < axes && i < 4; ++i) at.sections[i] = sections[i];
    kernels::apply_rope_axes(tq, tk, at);
    return kernels::last_error().empty() ? 0 : -1;
}

// Calls with a tensor that does not fit; nothing is read.  Returns 0 where the call was not refused.
int bas_refusal(int op)
{
    void* const p = reinterpret_cast<void*>(uintptr_t{256});
    int* const  i = static_cast<int*>(p);
    auto gpu = [&](std::vector<int64_t> s, DType t = DType::BF16) { return Tensor::from_external(p, std::move(s), t, Device::GPU); };
    Tensor q = gpu({2, 1, 4, 64}), k = gpu({2, 1, 2, 64}), c = gpu({4, 16, 2, 64}), c8 = gpu({4, 16, 2, 64}, DType::I8);
    Tensor box = gpu({4, 2, 2, 64}), li = gpu({2, 1, 2, 3}, DType::I32), o = gpu({2, 1, 256}), half = gpu({2, 1, 2, 64}, DType::F16);
    Tensor wide = gpu({4, 32, 2, 64}), few = gpu({2, 1, 1, 3}, DType::I32), small = gpu({1, 1, 256}), f32 = gpu({4, 2, 2, 64}, DType::F32);
    kernels::AxisPositions at{};
    at.positions = i;
    at.axes = 2;
    at.sections[0] = at.sections[1] = 16;
    kernels::AxisPositions off = at;
    off.sections[1] = 15;
    switch (op)
    {
        case -1: kernels::update_key_bounds(c, box, i, i, 0, 2, 1); break;  // no rows: nothing to refuse
        case 0: kernels::apply_rope_axes(half, k, at); break;
        case 1: kernels::apply_rope_axes(q, k, off); break;
        case 2: kernels::rope_append_kv_cache_axes(q, k, half, c, c, i, i, 2, at); break;
        case 3: kernels::rope_append_kv_cache_axes(q, k, k, wide, wide, i, i, 2, at); break;
        case 4: kernels::rope_append_kv_cache_axes(q, k, k, c8, c8, i, i, 2, at); break;
        case 5: kernels::rope_append_kv_cache_axes(q, k, k, c, c, i, i, 2, at, nullptr, nullptr, &k); break;
        case 6: kernels::update_key_bounds(c, f32, i, i, 2, 2, 1); break;
        case 7: kernels::update_key_bounds(wide, box, i, i, 2, 2, 1); break;
        case 8: kernels::update_key_bounds(c8, box, i, i, 2, 2, 1); break;
        case 9: kernels::select_blocks(q, box, few, i, i, 9, 1, 1); break;
        case 10: kernels::select_blocks(q, c, li, i, i, 9, 1, 1); break;
        case 11: kernels::select_blocks(q, box, li, i, i, 9, 2, 2); break;
        case 12: kernels::select_blocks(q, box, li, i, i, 9, 1, 1, 0); break;
        case 13: kernels::attention_blocks(q, c, c, o, few, i, i, 9); break;
        case 14: kernels::attention_blocks(q, c, c, small, li, i, i, 9); break;
        case 15: kernels::attention_blocks(q, wide, wide, o, li, i, i, 9); break;
        case 16: kernels::attention_blocks(q, c8, c8, o, li, i, i, 9); break;
        default: kernels::attention_blocks(q, c, c8, o, li, i, i, 9);
    }
    return kernels::last_error().empty() ? 0 : -1;
}

}  // extern "C"
