// capi_util.h - what the C ABI's translation units share: the calling thread's error message, checks of arguments, and
// the decode's workspace layout.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>

#include "ffkv.h"
#include "ffkv_internal.h"

namespace ffkv::capi
{

inline thread_local std::string g_last_error;

inline int fail(int code, const char* fmt, ...)
{
    char    buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_last_error = buf;
    return code;
}

inline int ok()
{
    g_last_error.clear();
    return FFKV_OK;
}

inline int hip_fail(hipError_t e, const char* what)
{
    return fail(FFKV_ERR_HIP, "%s: %s (%d)", what, hipGetErrorString(e), static_cast<int>(e));
}

// Whether `s` is being captured; FFKV_OK or the error.  The library allocates no stream-ordered memory inside a capture: a
// graph of three calls that each allocated and freed their own faulted on its first replay.
inline int is_capturing(hipStream_t s, bool& yes)
{
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const hipError_t       e = hipStreamIsCapturing(s, &status);
    yes = status != hipStreamCaptureStatusNone;
    return e == hipSuccess ? FFKV_OK : hip_fail(e, "hipStreamIsCapturing");
}

inline bool is_act(int dt) { return dt == FFKV_DTYPE_F32 || dt == FFKV_DTYPE_F16 || dt == FFKV_DTYPE_BF16; }
inline bool is_cache(int dt) { return is_act(dt) || dt == FFKV_DTYPE_I8 || dt == FFKV_DTYPE_FP8_E4M3; }
inline bool quantized(int dt) { return dt == FFKV_DTYPE_I8 || dt == FFKV_DTYPE_FP8_E4M3; }
// Append and decode take any head_dim that is a multiple of 8 up to 128 (as the reference's decode, one 8-element
// vector per lane of a 16-lane group: src/kernels/attention.cu:307-316), and 256; prefill and rope+append take 64,
// 128 and 256 (the reference's prefill and rope take 128, and 64 / 128).
inline bool head_dim_ok(int d) { return d == 256 || (d >= 8 && d <= 128 && d % 8 == 0); }
inline bool head_dim_mfma(int d) { return d == 64 || d == 128 || d == 256; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace ffkv::capi

namespace ffkv
{

// MFMA workspace layout: [row meta: batch x 2 int32 | (m, l): slots x num_heads x 2 fp32 | acc: slots x num_heads
// x head_dim fp32], each region 256-byte aligned, slots = items + batch (slot = work item + row) plus, in
// shared-prefix mode, prefix_chunks slots per row after those.  The public size query assumes kMfmaMaxItems items.
struct MfmaLayout
{
    int64_t meta, ml, acc, total;
};

MfmaLayout mfma_layout(int batch, int num_heads, int head_dim, int prefix_chunks = 0, int items = kMfmaMaxItems);
int        decode_most_items(int batch, int cap_tokens);

}  // namespace ffkv
