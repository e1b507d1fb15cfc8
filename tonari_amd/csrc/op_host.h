// What the C ABI of the operators shares on the host: checks of requests and the
// choice of an instance by type.
#pragma once

#include "op_common.h"

#include <cstdio>

namespace tnr {
namespace op {

inline int refuse(char* err, size_t len, const char* message) {
    if (err && len) std::snprintf(err, len, "%s", message);
    return TNR_INPUT_ERROR;
}

inline int launched(char* err, size_t len) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return TNR_OK;
    if (err && len) std::snprintf(err, len, "HIP error: %s", hipGetErrorString(e));
    return TNR_DEVICE_ERROR;
}

inline bool is_type(int32_t dtype) {
    return dtype == TNR_FLOAT32 || dtype == TNR_BFLOAT16 || dtype == TNR_FLOAT16;
}
inline size_t size_of(int32_t dtype) { return dtype == TNR_FLOAT32 ? 4 : 2; }
inline size_t padded(size_t bytes) { return (bytes + 255) / 256 * 256; }

template <typename F>
void with_type(int32_t dtype, F&& f) {
    if (dtype == TNR_FLOAT32)
        f(float{});
    else if (dtype == TNR_BFLOAT16)
        f(bf16{});
    else
        f(f16{});
}
template <int N>
struct Int {
    static constexpr int value = N;
};

// A launch of more than 2^32 threads is not possible.
constexpr int64_t kMostThreads = (int64_t(1) << 32) - 1;

// ------------------------------------------------------------------ attention

inline int check_heads(int32_t dtype, int32_t heads, int32_t kv_heads, int32_t dim, float scale,
                float softcap, char* err, size_t len) {
    if (!is_type(dtype)) return refuse(err, len, "dtype must be float32, bfloat16 or float16");
    if (heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || heads > 1024)
        return refuse(err, len, "heads must be a multiple of the key and value heads, at most 1024");
    if (dim < 8 || dim > 128 || dim % 8 != 0)
        return refuse(err, len, "the head dimension must be a multiple of 8, from 8 to 128");
    if (!std::isfinite(scale)) return refuse(err, len, "scale must be finite");
    if (!std::isfinite(softcap) || softcap < 0.f)
        return refuse(err, len, "softcap must be finite and positive");
    const ScoreRule rule = ScoreRule::of(scale, softcap);
    if (!std::isfinite(rule.scale2) || !std::isfinite(rule.inv) || !std::isfinite(rule.cap2))
        return refuse(err, len, "scale, softcap or scale / softcap is too large for 32 bits");
    return TNR_OK;
}

// Rows of a tile are found by 32-bit offsets.
constexpr int64_t kMostStride = int64_t(1) << 24;
inline bool aligned(const void* p, const int64_t (&stride)[2], int32_t dtype) {
    const int64_t unit = 16 / (int64_t)size_of(dtype);
    for (const int64_t s : stride)
        if (s % unit != 0 || s < 0 || s > kMostStride) return false;
    return (uintptr_t)p % 16 == 0;
}

}  // namespace op
}  // namespace tnr
