// rn_cache.hip — keys and values quantised into a caller-held cache as they are
// written, and read back (rn_cache_write, rn_cache_read).
//
// A row x of 64 values: peak = max |x|, scale = peak / 127 (1 where the peak is not
// positive), code = clamp(round-half-even(x / scale)): ops::quantise_int8
// (ops.rs:103-118) bit for bit, so that a cache written here is the cache the int8
// sessions hold. Read back: code * scale, one rounding.
//
// Both kernels only move memory. Eight lanes hold a row (16 bytes of fp16, 32 of
// f32, 8 of codes a lane), so that a wave's eight rows, consecutive tokens of one
// head, are one contiguous run of the cache (512 bytes of codes) and eight
// 256-byte runs of the caller's rows; the scale's few operations are shared by
// eight values a lane. A wave takes keys and values together: four 16-byte loads of
// f32 in flight a lane.
#include "rn_device.hpp"
#include "rn_serving.hpp"

namespace rn {
namespace {

constexpr int kRowLanes = 8;                       // lanes a row
constexpr int kLaneValues = kCacheWidth / kRowLanes;
constexpr int kWaveTokens = kWave / kRowLanes;     // tokens a wave takes at once

struct CacheMove {
    CacheDev cache;
    char* keys;     // the caller's rows
    char* values;
    int64_t sequence_stride, token_stride, head_stride;  // elements
    const int32_t* starts;
    const int32_t* counts;
    int32_t* error;
    int tokens, tiles;  // tiles: waves a (sequence, head)
};

// This wave's (sequence, head, first token), and where the sequence's rows go.
// False where there is nothing to move.
__device__ __forceinline__ bool cache_place(const CacheMove& p, int64_t& row, int64_t& source, int& left) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(blockIdx.x * (blockDim.x / kWave) + threadIdx.x / kWave);
    const uint32_t pair = wave / (uint32_t)p.tiles, tile = wave - pair * (uint32_t)p.tiles;
    const int sequence = (int)(pair / (uint32_t)p.cache.kv_heads), head = (int)(pair - sequence * p.cache.kv_heads);
    if (sequence >= p.cache.sequences) return false;
    const int start = p.starts ? p.starts[sequence] : 0, count = p.counts ? p.counts[sequence] : p.tokens;
    if (start < 0 || count < 0 || count > p.tokens || start > p.cache.capacity - count) {
        if (p.error && tile == 0 && head == 0 && threadIdx.x % kWave == 0) *p.error = RN_ERR_ARGUMENT;
        return false;
    }
    const int token = (int)tile * kWaveTokens;
    left = count - token;
    row = sequence * p.cache.sequence_rows + head * p.cache.head_rows + start + token;
    source = sequence * p.sequence_stride + head * p.head_stride + token * p.token_stride;
    return left > 0;
}

template <typename T>
__device__ __forceinline__ void load_row(const T* src, float* v) {
    if constexpr (sizeof(T) == 4) {
        load_floats<kLaneValues>(src, v);
    } else {
        const uint4 t = *reinterpret_cast<const uint4*>(src);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __half2float(__ushort_as_half((unsigned short)(w[i] & 0xffffu)));
            v[2 * i + 1] = __half2float(__ushort_as_half((unsigned short)(w[i] >> 16)));
        }
    }
}

__device__ __forceinline__ uint32_t two_halves(float a, float b) {
    return (uint32_t)__half_as_ushort(__float2half_rn(a)) | ((uint32_t)__half_as_ushort(__float2half_rn(b)) << 16);
}

template <typename T>
__device__ __forceinline__ void store_row(T* dst, const float* v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(dst) = make_uint4(two_halves(v[0], v[1]), two_halves(v[2], v[3]),
                                                    two_halves(v[4], v[5]), two_halves(v[6], v[7]));
    }
}

// One row's eight values a lane to codes and their scale.
__device__ __forceinline__ uint2 quantise_row(const float* v, float& scale) {
    float peak = 0.0f;
#pragma unroll
    for (int i = 0; i < kLaneValues; ++i) peak = fmaxf(peak, fabsf(v[i]));
    uint32_t u = __float_as_uint(peak);  // not negative, no NaN: ordered as its bits are
    u = max(u, (uint32_t)dpp_move<0xb1>((int)u));
    u = max(u, (uint32_t)dpp_move<0x4e>((int)u));
    u = max(u, (uint32_t)dpp_move<0x141>((int)u));
    scale = int8_scale_from_peak(__uint_as_float(u));
    float y[kLaneValues];
    quotients<kLaneValues>(v, scale, y);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < kLaneValues; ++i) w[i / 4] |= ((uint32_t)code_of_quotient(y[i]) & 0xffu) << (8 * (i % 4));
    return make_uint2(w[0], w[1]);
}

template <typename T, bool I8>
__global__ __launch_bounds__(256) void cache_write_kernel(const CacheMove p) {
    int64_t row, source;
    int left;
    if (!cache_place(p, row, source, left)) return;
    const int lane = threadIdx.x % kWave, token = lane / kRowLanes, at = (lane % kRowLanes) * kLaneValues;
    // lanes past the count read the last row again (every lane takes part in the
    // quantisation's vote) and store nothing
    const int64_t from = source + (token < left ? token : left - 1) * p.token_stride + at;
    float k[kLaneValues], v[kLaneValues];
    load_row(reinterpret_cast<const T*>(p.keys) + from, k);
    load_row(reinterpret_cast<const T*>(p.values) + from, v);
    const int64_t to = row + token;
    if constexpr (I8) {
        float ks, vs;
        const uint2 kc = quantise_row(k, ks), vc = quantise_row(v, vs);
        if (token >= left) return;
        *reinterpret_cast<uint2*>(p.cache.keys + to * kCacheWidth + at) = kc;
        *reinterpret_cast<uint2*>(p.cache.values + to * kCacheWidth + at) = vc;
        if (at == 0) {
            p.cache.key_scales[to] = ks;
            p.cache.value_scales[to] = vs;
        }
    } else {
        if (token >= left) return;
        store_row(reinterpret_cast<__half*>(p.cache.keys) + to * kCacheWidth + at, k);
        store_row(reinterpret_cast<__half*>(p.cache.values) + to * kCacheWidth + at, v);
    }
}

__device__ __forceinline__ void codes_row(uint2 codes, float scale, float* v) {
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < kLaneValues; ++i) {
        v[i] = (float)(int)(int8_t)(w[i / 4] >> (8 * (i % 4))) * scale;
        // the product is rounded to f32 whatever it is stored as: without this the
        // compiler folds it and the conversion to fp16 into one v_fma_mixlo_f16
        asm("" : "+v"(v[i]));
    }
}

template <typename T, bool I8>
__global__ __launch_bounds__(256) void cache_read_kernel(const CacheMove p) {
    int64_t row, source;
    int left;
    if (!cache_place(p, row, source, left)) return;
    const int lane = threadIdx.x % kWave, token = lane / kRowLanes, at = (lane % kRowLanes) * kLaneValues;
    if (token >= left) return;
    const int64_t from = row + token, to = source + token * p.token_stride + at;
    float k[kLaneValues], v[kLaneValues];
    if constexpr (I8) {
        const uint2 kc = *reinterpret_cast<const uint2*>(p.cache.keys + from * kCacheWidth + at);
        const uint2 vc = *reinterpret_cast<const uint2*>(p.cache.values + from * kCacheWidth + at);
        const float ks = p.cache.key_scales[from], vs = p.cache.value_scales[from];
        codes_row(kc, ks, k);
        codes_row(vc, vs, v);
    } else {
        load_row(reinterpret_cast<const __half*>(p.cache.keys) + from * kCacheWidth + at, k);
        load_row(reinterpret_cast<const __half*>(p.cache.values) + from * kCacheWidth + at, v);
    }
    store_row(reinterpret_cast<T*>(p.keys) + to, k);
    store_row(reinterpret_cast<T*>(p.values) + to, v);
}

int cache_move(const rn_cache* cache, const rn_cache_rows* rows, int tokens, const int32_t* starts,
               const int32_t* counts, int32_t* error, void* stream, bool write) {
    SV_CHECK(check_cache(cache, "cache"));
    SV_REQUIRE(rows, "rows is null");
    SV_REQUIRE(rows->type == RN_F32 || rows->type == RN_F16, "unknown element type %d", rows->type);
    SV_REQUIRE(tokens >= 0 && tokens <= cache->capacity, "tokens must be 0..%d (got %d)", cache->capacity, tokens);
    if (tokens == 0) return RN_OK;
    SV_REQUIRE(rows->keys && rows->values, "null rows");
    const int size = rows->type == RN_F32 ? 4 : 2, unit = rows->type == RN_F32 ? 4 : 8;
    const int64_t strides[3] = {rows->sequence_stride, rows->token_stride, rows->head_stride};
    const int64_t counted[3] = {cache->sequences, tokens, cache->kv_heads};
    for (int64_t s : strides)
        SV_REQUIRE(s >= 0 && s <= ((int64_t)1 << 40) && s % unit == 0,
                   "row strides must be whole multiples of 16 bytes, not negative");
    SV_REQUIRE(write || disjoint(kCacheWidth, strides, counted), "the rows to fill overlap");
    OnDevice on;
    SV_CHECK(on.enter((hipStream_t)stream));
    SV_CHECK(check_cache_pointers(on, cache));
    SV_CHECK(on.pointer(rows->keys, 16, "keys"));
    SV_CHECK(on.pointer(rows->values, 16, "values"));
    SV_CHECK(on.optional(starts, 4, "starts"));
    SV_CHECK(on.optional(counts, 4, "counts"));
    SV_CHECK(on.optional(error, 4, "error"));
    CacheMove p{cache_dev(cache), (char*)rows->keys, (char*)rows->values, strides[0], strides[1], strides[2],
                starts, counts, error, tokens, (tokens + kWaveTokens - 1) / kWaveTokens};
    const int64_t waves = (int64_t)cache->sequences * cache->kv_heads * p.tiles;
    SV_REQUIRE(waves <= ((int64_t)1 << 31), "too many rows for one call");
    const dim3 grid((uint32_t)((waves + 3) / 4)), block(256);
    const bool i8 = cache->format == RN_CACHE_I8;
    hipStream_t s = (hipStream_t)stream;
    if (write) {
        if (size == 4)
            rn_launch(i8 ? cache_write_kernel<float, true> : cache_write_kernel<float, false>, grid, block, 0, s, p);
        else
            rn_launch(i8 ? cache_write_kernel<__half, true> : cache_write_kernel<__half, false>, grid, block, 0, s, p);
    } else {
        if (size == 4)
            rn_launch(i8 ? cache_read_kernel<float, true> : cache_read_kernel<float, false>, grid, block, 0, s, p);
        else
            rn_launch(i8 ? cache_read_kernel<__half, true> : cache_read_kernel<__half, false>, grid, block, 0, s, p);
    }
    SV_HIP(hipGetLastError());
    return RN_OK;
}

}  // namespace
}  // namespace rn

using namespace rn;

int rn_cache_write(const rn_cache* cache, const rn_cache_rows* rows, int tokens, const int32_t* starts,
                   const int32_t* counts, int32_t* error, void* stream) {
    return cache_move(cache, rows, tokens, starts, counts, error, stream, true);
}

int rn_cache_read(const rn_cache* cache, const rn_cache_rows* rows, int tokens, const int32_t* starts,
                  const int32_t* counts, int32_t* error, void* stream) {
    return cache_move(cache, rows, tokens, starts, counts, error, stream, false);
}
