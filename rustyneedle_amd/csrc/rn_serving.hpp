// rn_serving.hpp — what the serving operators over caller-held memory share
// (rn_cache.hip, rn_shared.hip, rn_verify.hip): the checks of their arguments and
// the cache descriptor as the kernels take it.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/rustyneedle.h"
#include "rn_internal.hpp"

#define SV_REQUIRE(cond, ...)                                                    \
    do {                                                                         \
        if (!(cond)) return rn::serving_error(RN_ERR_ARGUMENT, __VA_ARGS__);     \
    } while (0)
#define SV_HIP(call)                                                             \
    do {                                                                         \
        hipError_t e_ = (call);                                                  \
        if (e_ != hipSuccess) {                                                  \
            (void)hipGetLastError();                                             \
            return rn::serving_error(RN_ERR_DEVICE, "%s: %s", #call, hipGetErrorString(e_)); \
        }                                                                        \
    } while (0)
#define SV_CHECK(call)                                                           \
    do {                                                                         \
        int rc_ = (call);                                                        \
        if (rc_ != RN_OK) return rc_;                                            \
    } while (0)

namespace rn {

constexpr int kCacheWidth = 64;  // values of a cache row

inline size_t aligned_bytes(size_t v) { return (v + 255) & ~(size_t)255; }

__attribute__((format(printf, 2, 3))) inline int serving_error(int code, const char* fmt, ...) {
    char text[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    return set_error(code, text);
}

// A cache as the kernels take it: row (sequence, head, position) is row number
// sequence * sequence_rows + head * head_rows + position of keys and values, and of
// the scales.
struct CacheDev {
    char* keys;
    char* values;
    float* key_scales;
    float* value_scales;
    int64_t sequence_rows, head_rows;
    int sequences, kv_heads, capacity;
};

inline CacheDev cache_dev(const rn_cache* c) {
    return {(char*)c->keys, (char*)c->values, c->key_scales, c->value_scales, c->sequence_rows, c->head_rows,
            c->sequences, c->kv_heads, c->capacity};
}

// The launches of a call go to the device of its stream (the current one for the
// default stream), and its pointers are looked at against that device: a host
// array or another device's memory is refused instead of faulting in a kernel
// (about 0.06 us a pointer).
class OnDevice {
public:
    int enter(hipStream_t stream) {
        SV_HIP(hipGetDevice(&before_));
        device_ = before_;
        if (stream != nullptr && stream != hipStreamPerThread && stream != hipStreamLegacy) {
            hipDevice_t d;
            SV_HIP(hipStreamGetDevice(stream, &d));
            device_ = (int)d;
        }
        if (device_ != before_) {
            SV_HIP(hipSetDevice(device_));
            moved_ = true;
        }
        return RN_OK;
    }
    ~OnDevice() {
        if (moved_) (void)hipSetDevice(before_);
    }
    int pointer(const void* p, size_t align, const char* name) const {
        SV_REQUIRE(((uintptr_t)p & (align - 1)) == 0, "%s must be aligned to %zu bytes", name, align);
        hipPointerAttribute_t at{};
        if (hipPointerGetAttributes(&at, p) != hipSuccess) {
            (void)hipGetLastError();
            return serving_error(RN_ERR_ARGUMENT, "%s is not device memory", name);
        }
        SV_REQUIRE(at.type == hipMemoryTypeDevice || at.type == hipMemoryTypeHost || at.type == hipMemoryTypeManaged,
                   "%s is not device memory", name);
        SV_REQUIRE(at.type != hipMemoryTypeDevice || at.device == device_,
                   "%s lies on device %d, the call's stream on device %d", name, at.device, device_);
        return RN_OK;
    }
    int optional(const void* p, size_t align, const char* name) const {
        return p == nullptr ? RN_OK : pointer(p, align, name);
    }

private:
    int before_ = 0, device_ = 0;
    bool moved_ = false;
};

// Whether elements at i*s0 + j*s1 + k*s2 (i < n0, ...; each `extent` long) never
// overlap: ordered by stride, each stride passes over everything inside it.
inline bool disjoint(int64_t extent, const int64_t strides[3], const int64_t counts[3]) {
    int order[3] = {0, 1, 2};
    for (int a = 0; a < 3; ++a)
        for (int b = a + 1; b < 3; ++b)
            if (strides[order[b]] < strides[order[a]]) {
                const int t = order[a];
                order[a] = order[b];
                order[b] = t;
            }
    int64_t inside = extent;  // from the first element of an inner run to past its last
    for (int a = 0; a < 3; ++a) {
        const int i = order[a];
        if (counts[i] <= 1) continue;
        if (strides[i] < inside) return false;
        int64_t steps;
        if (__builtin_mul_overflow(strides[i], counts[i] - 1, &steps)) return false;
        if (__builtin_add_overflow(inside, steps, &inside)) return false;
    }
    return true;
}

// The host's checks of a cache descriptor (no device call).
inline int check_cache(const rn_cache* c, const char* name) {
    SV_REQUIRE(c, "%s is null", name);
    SV_REQUIRE(c->format == RN_CACHE_F16 || c->format == RN_CACHE_I8, "%s: unknown cache format %d", name, c->format);
    SV_REQUIRE(c->sequences >= 1 && c->kv_heads >= 1 && c->capacity >= 1,
               "%s: sequences, kv_heads and capacity must be positive", name);
    SV_REQUIRE(c->sequences <= 65535 && c->kv_heads <= 1024 && c->capacity <= (1 << 24),
               "%s: at most 65535 sequences, 1024 heads and 2^24 positions", name);
    SV_REQUIRE(c->sequence_rows >= 0 && c->sequence_rows <= ((int64_t)1 << 40) && c->head_rows >= 0 &&
                   c->head_rows <= ((int64_t)1 << 40),
               "%s: bad strides", name);
    const int64_t strides[3] = {c->sequence_rows, c->head_rows, 1}, counts[3] = {c->sequences, c->kv_heads, c->capacity};
    SV_REQUIRE(disjoint(1, strides, counts), "%s: its sequences and heads overlap", name);
    SV_REQUIRE(c->keys && c->values, "%s: null keys or values", name);
    SV_REQUIRE(c->format == RN_CACHE_F16 || (c->key_scales && c->value_scales), "%s: an 8-bit cache needs scales",
               name);
    return RN_OK;
}

inline int check_cache_pointers(const OnDevice& on, const rn_cache* c) {
    SV_CHECK(on.pointer(c->keys, 16, "cache keys"));
    SV_CHECK(on.pointer(c->values, 16, "cache values"));
    if (c->format == RN_CACHE_I8) {
        SV_CHECK(on.pointer(c->key_scales, 4, "key scales"));
        SV_CHECK(on.pointer(c->value_scales, 4, "value scales"));
    }
    return RN_OK;
}

}  // namespace rn
