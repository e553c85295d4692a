// rn_shared.hip — attention of a batch over one shared prefix and each sequence's
// own cache (rn_attend_shared).
//
// For a query q of a (sequence, token, head), with c = scale log2(e):
//     s_k = q . k_k,  w_k = 2^(c s_k - m),  out = sum w_k v_k / sum w_k,
// over the positions the query sees; any m gives the same value, and the running
// maximum of c s_k keeps every w_k in range. The keys are split over blocks; each
// block leaves (m, sum w_k, sum w_k v_k) of its share, and one more launch joins the
// shares, each times 2^(m - max m).
//
// The rows of a block are queries: of every sequence for a share of the prefix (so
// the prefix is read once for all), of one sequence for a share of its own cache.
// v_mfma_f32_16x16x32_f16 computes scores with keys as rows and queries as columns,
// so a lane holds scores of one query, and they are the second product's B operand
// (keys x queries, against values transposed by ds_read_b64_tr_b16) as they are: its
// k slots may name the keys in any order as long as both operands agree.
//
// Precision: int8 codes and fp16 keys are exact in fp16. A query is scaled by a power
// of two (exact) to a peak in [2^13, 2^14) and enters as two fp16 numbers, hi + lo =
// 22 bits; a weight (times the value row's scale, over a power of two that bounds
// those scales) likewise. Each product is so twice the matrix instructions of a
// single fp16 one, with f32 sums: about 1e-6 from the exact value where a single one
// is off by 2e-4.
#include "rn_device.hpp"
#include "rn_serving.hpp"

namespace rn {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;       // keys a tile
constexpr int kWeightBits = 14;  // weights are held times 2^14: small ones keep their bits as fp16 pairs
constexpr int kStageBytes = 2 * kTile * kCacheWidth * 2 + 2 * kTile * 4;  // keys, values as fp16, scales

struct SharedParams {
    const float* q;
    float* out;
    int64_t q_stride, out_stride;
    CacheDev prefix, own;  // own.capacity 0: none
    const int32_t* lengths;
    const int32_t* counts;
    float* parts;   // [slots][rows][64]
    float2* stats;  // [slots][rows]: the reference (log2) and the sum of weights
    int32_t* error;
    int sequences, queries, kv_heads, group, rows;
    int prefix_first, prefix_length, window;
    int prefix_tiles, prefix_splits, prefix_tasks, own_tiles, own_splits;
    float scale2;  // scale log2(e)
};

struct Sequence {
    int length, count;
    bool bad;
};
__device__ __forceinline__ Sequence sequence_of(const SharedParams& p, int b) {
    Sequence s;
    s.length = p.lengths ? p.lengths[b] : p.own.capacity;
    s.count = p.counts ? p.counts[b] : p.queries;
    s.bad = s.length < 0 || s.length > p.own.capacity || s.count < 0 || s.count > p.queries;
    if (s.bad) s.length = s.count = 0;
    return s;
}

// max(a, b) without the canonicalising moves of fmaxf; NaN loses to a number.
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_fmaxf(a, b); }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// Four int8 codes as fp16: the byte c ^ 0x80 = c + 128 under the exponent of 1024 is
// 1152 + c exactly; less 1152.
__device__ __forceinline__ void halves_of_codes(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u);
    const v2h bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, a) - bias);
    hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, b) - bias);
}

// Where the 16-byte chunk `chunk` (0..7) of key row `row` lies in a staged tile:
// rows are 128 bytes, the chunks of eight rows in a row permuted so that the sixteen
// lanes that read one chunk of sixteen rows meet different banks.
__device__ __forceinline__ int staged(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// Both fp16 parts of two numbers: hi + lo = 22 bits of each.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
    typedef __fp16 v2f __attribute__((ext_vector_type(2)));
    const v2f h = __builtin_amdgcn_cvt_pkrtz(a, b);
    const v2f l = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h[0], -1.0f, a), __builtin_fmaf((float)h[1], -1.0f, b));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

union Frag {
    uint32_t w[4];
    uint4 q;
    v8h h;
};

__device__ __forceinline__ v4f mfma(const Frag& a, const Frag& b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
}

// A share of the keys for 16 QT WM query rows. Four waves: WM of them hold different
// rows and share each staged tile, the 4 / WM groups take tiles in turn and are
// joined at the end. Waves of a group of one stage for themselves, without barriers.
template <bool I8, int QT, int WM>
struct Job {
    static constexpr int kGroups = 4 / WM, kRows = 16 * QT * WM, kThreads = 64 * WM;
    static constexpr int kChunks = (I8 ? 4 : 8) * kTile / kThreads;  // 16-byte loads a thread, keys and values each

    struct Row {
        int lo, hi;   // the local positions this row sees
        int id;       // row number in out and the partials, -1: none
        float rs;     // c over the query's scaling
        float m, mr;  // running maximum of the raw scores, and times rs
        float l;      // this lane's share of the sum of weights
    };

    const SharedParams& p;
    char* lds;
    const int lane, col, quad, wave, wm, wk, thread;

    __device__ Job(const SharedParams& p_, char* lds_)
        : p(p_), lds(lds_), lane(threadIdx.x % 64), col(lane % 16), quad(lane / 16), wave(threadIdx.x / 64),
          wm(wave % WM), wk(wave / WM), thread(threadIdx.x % kThreads) {}

    __device__ __forceinline__ void sync() const {
        if constexpr (WM == 1)
            wave_lds_sync();
        else
            __syncthreads();
    }

    __device__ void run(const CacheDev& cache, bool prefix, int sequence, int head, int tile, int split, int splits,
                        int slot) {
        const int T = p.queries, G = p.group, P = p.prefix_length;
        // ---- the rows and their queries
        Row row[QT];
        Frag qh[QT][2], ql[QT][2];
        int lo_most = 0, hi_least = 0x7fffffff;
        int first, last;  // this share's keys come from [first, last)
        if (prefix) {
            first = p.prefix_first;
            last = P;
        } else {
            const Sequence s = sequence_of(p, sequence);
            const int seen = P + s.length - s.count + 1 - p.window;  // the first query's first position
            first = p.window > 0 && seen > P ? min(seen - P, s.length) : 0;
            last = s.length;
        }
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            const int r = tile * kRows + (wm * QT + i) * 16 + col;
            Row& w = row[i];
            w.id = -1;
            w.lo = 0;
            w.hi = 0x7fffffff;
            const float* q = nullptr;
            if (r < (prefix ? p.sequences : 1) * T * G) {
                const int b = prefix ? r / (T * G) : sequence, in = prefix ? r - b * T * G : r;
                const int t = in / G, g = in - t * G;
                const Sequence s = sequence_of(p, b);
                if (t < s.count) {
                    w.id = (b * T + t) * p.kv_heads * G + head * G + g;
                    q = p.q + (int64_t)(b * T + t) * p.q_stride + (head * G + g) * kCacheWidth;
                    const int end = P + s.length - s.count + t + 1;
                    const int begin = p.window > 0 ? max(end - p.window, 0) : 0;
                    w.hi = prefix ? end : end - P;
                    w.lo = prefix ? begin : begin - P;
                    lo_most = max(lo_most, w.lo);
                    hi_least = min(hi_least, w.hi);
                }
            }
            float v[2][8];
            float peak = 0.0f;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[s][j] = 0.0f;
                if (q) load_floats<8>(q + 32 * s + 8 * quad, v[s]);
#pragma unroll
                for (int j = 0; j < 8; ++j) peak = max_of(peak, fabsf(v[s][j]));
            }
            peak = max_of(peak, lane_xor<16>(peak));
            peak = max_of(peak, lane_xor<32>(peak));
            const int e = peak < __builtin_inff() ? (int)(__float_as_uint(peak) >> 23) - 127 : 0;
            w.rs = max_of(__builtin_ldexpf(p.scale2, e - 13), 0x1p-126f);
            w.m = -__builtin_inff();
            w.mr = 0.0f;
            w.l = 0.0f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    split_pair(__builtin_ldexpf(v[s][2 * j], 13 - e), __builtin_ldexpf(v[s][2 * j + 1], 13 - e),
                               qh[i][s].w[j], ql[i][s].w[j]);
        }
        // the least and most over the wave's rows
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) {
            lo_most = max(lo_most, __shfl_xor(lo_most, x));
            hi_least = min(hi_least, __shfl_xor(hi_least, x));
        }
        lo_most = __builtin_amdgcn_readfirstlane(lo_most);
        hi_least = __builtin_amdgcn_readfirstlane(hi_least);

        // ---- the share's tiles
        const int tiles = (last - first + kTile - 1) / kTile;
        const int t0 = (int)((int64_t)tiles * split / splits), t1 = (int)((int64_t)tiles * (split + 1) / splits);
        const int64_t base = (prefix ? 0 : (int64_t)sequence * cache.sequence_rows) + (int64_t)head * cache.head_rows;
        const char* keys = cache.keys + base * (I8 ? 64 : 128);
        const char* values = cache.values + base * (I8 ? 64 : 128);
        const float* key_scales = I8 ? cache.key_scales + base : nullptr;
        const float* value_scales = I8 ? cache.value_scales + base : nullptr;
        char* stage = lds + wk * kStageBytes;
        char* stage_v = stage + kTile * 128;
        float* stage_ks = reinterpret_cast<float*>(stage + 2 * kTile * 128);
        float* stage_vs = stage_ks + kTile;

        v4f acc[QT][4];
#pragma unroll
        for (int i = 0; i < QT; ++i)
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[i][d] = v4f{0, 0, 0, 0};
        int bound = -200;  // acc is held over 2^bound (I8): every value scale so far is below 2^bound

        uint4 kr[kChunks], vr[kChunks];
        float ksr = 0.0f, vsr = 0.0f;
        constexpr int kRowChunks = I8 ? 4 : 8;
        auto fetch = [&](int t) {
            const int k0 = first + t * kTile;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int chunk = thread + c * kThreads, key = min(k0 + chunk / kRowChunks, last - 1);
                const int64_t at = (int64_t)key * (I8 ? 64 : 128) + chunk % kRowChunks * 16;
                kr[c] = *reinterpret_cast<const uint4*>(keys + at);
                vr[c] = *reinterpret_cast<const uint4*>(values + at);
            }
            if constexpr (I8) {
                if (thread < kTile) {
                    const int key = min(k0 + thread, last - 1);
                    ksr = key_scales[key];
                    vsr = value_scales[key];
                }
            }
        };
        auto put = [&](int t) {
            const int k0 = first + t * kTile;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int chunk = thread + c * kThreads, r = chunk / kRowChunks, part = chunk % kRowChunks;
                if constexpr (I8) {
                    uint4 a, b;
                    halves_of_codes(kr[c].x, a.x, a.y);
                    halves_of_codes(kr[c].y, a.z, a.w);
                    halves_of_codes(kr[c].z, b.x, b.y);
                    halves_of_codes(kr[c].w, b.z, b.w);
                    *reinterpret_cast<uint4*>(stage + staged(r, 2 * part)) = a;
                    *reinterpret_cast<uint4*>(stage + staged(r, 2 * part + 1)) = b;
                    halves_of_codes(vr[c].x, a.x, a.y);
                    halves_of_codes(vr[c].y, a.z, a.w);
                    halves_of_codes(vr[c].z, b.x, b.y);
                    halves_of_codes(vr[c].w, b.z, b.w);
                    *reinterpret_cast<uint4*>(stage_v + staged(r, 2 * part)) = a;
                    *reinterpret_cast<uint4*>(stage_v + staged(r, 2 * part + 1)) = b;
                } else {
                    // rows past the last hold zeros: a weight of 0 must not meet a NaN
                    const bool in = k0 + r < last;
                    *reinterpret_cast<uint4*>(stage + staged(r, part)) = kr[c];
                    *reinterpret_cast<uint4*>(stage_v + staged(r, part)) = in ? vr[c] : make_uint4(0, 0, 0, 0);
                }
            }
            if constexpr (I8) {
                if (thread < kTile) {
                    const bool in = k0 + thread < last;
                    stage_ks[thread] = in ? ksr : 0.0f;
                    stage_vs[thread] = in ? vsr : 0.0f;
                }
            }
        };

        const int rounds = (t1 - t0 + kGroups - 1) / kGroups;
        if (t0 + wk < t1) fetch(t0 + wk);
        for (int it = 0; it < rounds; ++it) {
            const int t = t0 + it * kGroups + wk;
            sync();  // the waves that read the tile before are done with it
            if (t < t1) put(t);
            sync();
            if (t + kGroups < t1) fetch(t + kGroups);
            if (t >= t1) continue;
            const int k0 = first + t * kTile;
            const bool masked = lo_most > k0 || min(hi_least, last) < k0 + kTile;
            v4f ks[4], vs[4];
            if constexpr (I8) {
                // the bound over the value scales
                float most = fabsf(stage_vs[lane]);
                most = wave_max_nonneg(most < __builtin_inff() ? most : 0.0f);
                const int e = (int)(__float_as_uint(most) >> 23) - 126;
                if (e > bound) {
#pragma unroll
                    for (int i = 0; i < QT; ++i)
#pragma unroll
                        for (int d = 0; d < 4; ++d)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[i][d][j] = __builtin_ldexpf(acc[i][d][j], bound - e);
                    bound = e;
                }
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    ks[kt] = *reinterpret_cast<const v4f*>(stage_ks + kt * 16 + quad * 4);
                    vs[kt] = *reinterpret_cast<const v4f*>(stage_vs + kt * 16 + quad * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) vs[kt][j] = __builtin_ldexpf(vs[kt][j], -bound);
                }
            }
            // ---- scores
            v4f s[QT][4];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                Frag a[2];
#pragma unroll
                for (int d = 0; d < 2; ++d)
                    a[d].q = *reinterpret_cast<const uint4*>(stage + staged(kt * 16 + col, d * 4 + quad));
#pragma unroll
                for (int i = 0; i < QT; ++i) {
                    v4f c = v4f{0, 0, 0, 0};
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        c = mfma(a[d], ql[i][d], c);
                        c = mfma(a[d], qh[i][d], c);
                    }
                    if constexpr (I8) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) c[j] *= ks[kt][j];
                    }
                    s[i][kt] = c;
                }
            }
            // ---- weights
            Frag wh[QT][2], wl[QT][2];
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                Row& w = row[i];
                if (masked) {
#pragma unroll
                    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = k0 + kt * 16 + quad * 4 + j;
                            if (key < w.lo || key >= w.hi || key >= last) s[i][kt][j] = -__builtin_inff();
                        }
                }
                float m = w.m;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) m = max_of(m, s[i][kt][j]);
                m = max_of(m, lane_xor<16>(m));
                m = max_of(m, lane_xor<32>(m));
                if (__any(m > w.m)) {
                    const float mr = m > w.m ? m * w.rs : w.mr;
                    const float alpha = w.m > -__builtin_inff() ? exp2_of(w.mr - mr) : 1.0f;  // 1: the sums are 0 yet
                    w.l *= alpha;
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][d][j] *= alpha;
                    w.m = m;
                    w.mr = mr;
                }
                const float c = (float)kWeightBits - w.mr;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    float x[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[j] = exp2_of(__builtin_fmaf(s[i][kt][j], w.rs, c));
                        w.l += x[j];
                        if constexpr (I8) x[j] *= vs[kt][j];
                    }
                    if (I8 && masked) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int key = k0 + kt * 16 + quad * 4 + j;
                            if (key < w.lo || key >= w.hi || key >= last) x[j] = 0.0f;
                        }
                    }
                    const int step = kt / 2, at = kt % 2 * 2;
                    split_pair(x[0], x[1], wh[i][step].w[at], wl[i][step].w[at]);
                    split_pair(x[2], x[3], wh[i][step].w[at + 1], wl[i][step].w[at + 1]);
                }
            }
            // ---- values
            typedef __attribute__((address_space(3))) v4s lds_v4s;
            bool odd = false;  // a masked tile of fp16 values holds an infinity or NaN
#pragma unroll
            for (int step = 0; step < 2; ++step)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    Frag a;
                    v4s part[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int r = step * 32 + x * 16 + quad * 4 + col / 4;
                        char* at = stage_v + staged(r, d * 2 + col % 4 / 2) + col % 2 * 8;
                        part[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
                    }
                    a.w[0] = __builtin_bit_cast(uint2, part[0]).x;
                    a.w[1] = __builtin_bit_cast(uint2, part[0]).y;
                    a.w[2] = __builtin_bit_cast(uint2, part[1]).x;
                    a.w[3] = __builtin_bit_cast(uint2, part[1]).y;
                    if (!I8 && masked) {
                        // left out here (0 x NaN is NaN) and added below to the rows that see them
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            uint32_t bad = 0;
                            if ((a.w[x] & 0x7c00u) == 0x7c00u) bad |= 0xffffu;
                            if ((a.w[x] & 0x7c000000u) == 0x7c000000u) bad |= 0xffff0000u;
                            odd = odd || bad;
                            a.w[x] &= ~bad;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < QT; ++i) {
                        acc[i][d] = mfma(a, wl[i][step], acc[i][d]);
                        acc[i][d] = mfma(a, wh[i][step], acc[i][d]);
                    }
                }
            if (!I8 && masked && __any(odd)) odd_values(row, s, acc, stage_v, k0, last);
        }
        finish(row, acc, bound, slot, prefix, sequence);
    }

    // The infinities and NaN of a masked tile's fp16 values, one key at a time, to the
    // rows that see the key.
    __device__ __forceinline__ void odd_values(const Row (&row)[QT], const v4f (&s)[QT][4], v4f (&acc)[QT][4],
                                               const char* stage_v, int k0, int last) const {
#pragma unroll 1
        for (int r = 0; r < kTile; ++r) {
            const int key = k0 + r;
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                float score = 0.0f;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) score = r / 16 == kt && r % 4 == j ? s[i][kt][j] : score;
                score = __shfl(score, r % 16 / 4 * 16 + col);
                const float x = exp2_of(__builtin_fmaf(score, row[i].rs, (float)kWeightBits - row[i].mr));
                const bool seen = key >= row[i].lo && key < row[i].hi && key < last;
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int at = d * 16 + quad * 4 + y;
                        const float v =
                            __half2float(*reinterpret_cast<const __half*>(stage_v + staged(r, at / 8) + at % 8 * 2));
                        if (seen && !(fabsf(v) < __builtin_inff())) acc[i][d][y] += x * v;
                    }
            }
        }
    }

    // A finished row quarter: partial sums, or the output where they are the only ones.
    __device__ __forceinline__ void leave(int id, int at, float4 o, float mr, float l, int slot) const {
        if (p.parts) {
            const int64_t r = (int64_t)slot * p.rows + id;
            if (at == 0) p.stats[r] = make_float2(mr, l);
            if (l != 0.0f) *reinterpret_cast<float4*>(p.parts + r * kCacheWidth + at) = o;
        } else {
            const int heads = p.kv_heads * p.group, token = id / heads;
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            *reinterpret_cast<float4*>(p.out + token * p.out_stride + (id - token * heads) * kCacheWidth + at) =
                make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        }
    }

    __device__ void finish(Row (&row)[QT], v4f (&acc)[QT][4], int bound, int slot, bool prefix, int sequence) const {
#pragma unroll
        for (int i = 0; i < QT; ++i) {
            row[i].l += lane_xor<16>(row[i].l);
            row[i].l += lane_xor<32>(row[i].l);
            if constexpr (I8) {
#pragma unroll
                for (int d = 0; d < 4; ++d)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][d][j] = __builtin_ldexpf(acc[i][d][j], bound);
            }
        }
        if constexpr (kGroups == 1) {
#pragma unroll
            for (int i = 0; i < QT; ++i)
                if (row[i].id >= 0) {
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        leave(row[i].id, d * 16 + quad * 4,
                              make_float4(acc[i][d][0], acc[i][d][1], acc[i][d][2], acc[i][d][3]), row[i].mr,
                              row[i].l, slot);
                }
        } else {
            // every wave's sums go to LDS: [wave][16 QT][64] and their (reference, sum, row)
            __syncthreads();
            float* sums = reinterpret_cast<float*>(lds);
            float4* heads = reinterpret_cast<float4*>(lds + 4 * 16 * QT * kCacheWidth * 4);
#pragma unroll
            for (int i = 0; i < QT; ++i) {
                const int r = wave * 16 * QT + i * 16 + col;
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<v4f*>(sums + r * kCacheWidth + (((d * 4 + quad) ^ col) << 2)) = acc[i][d];
                if (quad == 0) heads[r] = make_float4(row[i].mr, row[i].l, __int_as_float(row[i].id), 0.0f);
            }
            __syncthreads();
            for (int x = threadIdx.x; x < kRows * 16; x += 256) {
                const int r = x / 16, part = x % 16;
                const int in = r % (16 * QT), of = r / (16 * QT);  // row in its wave, wave of the group
                float4 h[kGroups];
                float m = -__builtin_inff();
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    h[k] = heads[(k * WM + of) * 16 * QT + in];
                    if (h[k].y != 0.0f) m = max_of(m, h[k].x);
                }
                const int id = __float_as_int(h[0].z);
                if (id < 0) continue;
                float4 o = make_float4(0, 0, 0, 0);
                float l = 0.0f;
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    if (h[k].y == 0.0f) continue;
                    const float a = exp2_of(h[k].x - m);
                    const float4 v = *reinterpret_cast<const float4*>(
                        sums + ((k * WM + of) * 16 * QT + in) * kCacheWidth + ((part ^ (in & 15)) << 2));
                    l += a * h[k].y;
                    o.x += a * v.x;
                    o.y += a * v.y;
                    o.z += a * v.z;
                    o.w += a * v.w;
                }
                leave(id, part * 4, o, l != 0.0f ? m : 0.0f, l, slot);
            }
        }
        // where nothing joins the shares, a sequence with bad numbers is answered here
        if (!p.parts && !prefix && sequence_of(p, sequence).bad) refuse(p, sequence);
    }

    static __device__ void refuse(const SharedParams& p, int sequence) {
        const int heads = p.kv_heads * p.group;
        for (int i = threadIdx.x; i < p.queries * heads * kCacheWidth; i += 256) {
            const int t = i / (heads * kCacheWidth);
            p.out[(int64_t)(sequence * p.queries + t) * p.out_stride + (i - t * heads * kCacheWidth)] = __builtin_nanf("");
        }
        if (p.error && threadIdx.x == 0) *p.error = RN_ERR_ARGUMENT;
    }
};

// Blocks 0..prefix_tasks-1: (key head, share, rows) of the prefix; the others:
// (sequence, key head, share, rows) of the own caches.
template <bool I8, int QP, int WP, int QO>
__global__ __launch_bounds__(256, 2) void shared_attend_kernel(const SharedParams p) {
    __shared__ __attribute__((aligned(16))) char lds[4 * kStageBytes];
    const int task = blockIdx.x;
    if (task < p.prefix_tasks) {
        const int tile = task % p.prefix_tiles, rest = task / p.prefix_tiles;
        const int split = rest % p.prefix_splits, head = rest / p.prefix_splits;
        Job<I8, QP, WP>(p, lds).run(p.prefix, true, 0, head, tile, split, p.prefix_splits, split);
    } else {
        int rest = task - p.prefix_tasks;
        const int tile = rest % p.own_tiles;
        rest /= p.own_tiles;
        const int split = rest % p.own_splits;
        rest /= p.own_splits;
        Job<I8, QO, 1>(p, lds).run(p.own, false, rest / p.kv_heads, rest % p.kv_heads, tile, split, p.own_splits,
                                   p.prefix_splits + split);
    }
}

// One wave a row of the output: the shares, each times 2^(its reference - the most).
// Sixteen lanes hold a row's 64 values, so a wave takes four shares at once; the loads
// of sixteen are in flight together (one share after the other, a lane a value, waits
// for every load: 20.8 us against 5.6 for 34 shares of 1920 rows).
__global__ __launch_bounds__(256) void shared_join_kernel(const SharedParams p) {
    const int id = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
    if (id >= p.rows) return;
    const int heads = p.kv_heads * p.group, token = id / heads;
    const int b = token / p.queries, at = lane % 16 * 4, quarter = lane / 16;
    const Sequence s = sequence_of(p, b);
    float* out = p.out + token * p.out_stride + (id - token * heads) * kCacheWidth;
    if (s.bad) {
        out[lane] = __builtin_nanf("");
        if (p.error && lane == 0) *p.error = RN_ERR_ARGUMENT;
        return;
    }
    if (token - b * p.queries >= s.count) return;
    const int slots = p.prefix_splits + p.own_splits;
    v4f o = v4f{0, 0, 0, 0};
    float l = 0.0f, most = -__builtin_inff();
    for (int k0 = 0; k0 < slots; k0 += 64) {
        const int mine = k0 + lane;
        const float2 st = mine < slots ? p.stats[(int64_t)mine * p.rows + id] : make_float2(0.0f, 0.0f);
        const float m = max_of(most, wave_max(st.y != 0.0f ? st.x : -__builtin_inff()));
        if (k0 > 0 && m > most) {
            const float a = exp2_of(most - m);
            l *= a;
            o *= a;
        }
        most = m;
        const float weight = st.y != 0.0f ? exp2_of(st.x - m) : 0.0f;
        l += weight * st.y;
        const int here = min(64, slots - k0);
        for (int k = 0; k < here; k += 16) {
            v4f v[4];
            float a[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int slot = k + 4 * u + quarter;
                a[u] = __shfl(weight, slot & 63);
                if (slot >= here) a[u] = 0.0f;
                v[u] = v4f{0, 0, 0, 0};
                if (a[u] != 0.0f)  // a share without weights holds nothing
                    v[u] = *reinterpret_cast<const v4f*>(p.parts + ((int64_t)(k0 + slot) * p.rows + id) * kCacheWidth + at);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) o += a[u] * v[u];
        }
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) l += __shfl_xor(l, m);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o[j] += lane_xor<16>(o[j]);
        o[j] += lane_xor<32>(o[j]);
    }
    if (quarter == 0) *reinterpret_cast<v4f*>(out + at) = l != 0.0f ? o / l : v4f{0, 0, 0, 0};
}

// How a call's rows and keys are dealt to blocks.
struct Plan {
    int rows = 0, qp = 1, wp = 1, qo = 1;  // row tiles: 16 qp wp rows of the prefix, 16 qo of an own cache
    int prefix_first = 0, prefix_tiles = 0, prefix_splits = 0, own_tiles = 0, own_splits = 0;
    size_t stats_at = 0, bytes = 0;
    bool direct = false;
};

constexpr int kBlocks = 512;  // blocks that fill the chip: two on each of 256 CUs

Plan plan_of(int sequences, int queries, int heads, int kv_heads, int prefix_length, int own_capacity, int window) {
    Plan n;
    const int group = heads / kv_heads;
    n.rows = sequences * queries * heads;
    const int shared_rows = sequences * queries * group, own_rows = queries * group;
    if (prefix_length > 0) {
        n.qp = shared_rows <= 16 ? 1 : 2;
        n.wp = shared_rows <= 32 ? 1 : shared_rows <= 64 ? 2 : 4;
        const int tile = 16 * n.qp * n.wp;
        n.prefix_tiles = (shared_rows + tile - 1) / tile;
        // no query sees below the first position of the first query of an empty own cache
        if (window > 0) n.prefix_first = prefix_length - queries + 1 - window > 0 ? prefix_length - queries + 1 - window : 0;
        if (n.prefix_first >= prefix_length) n.prefix_first = prefix_length - 1;
        const int keys = (prefix_length - n.prefix_first + kTile - 1) / kTile, most = (keys + 4 / n.wp - 1) / (4 / n.wp);
        const int base = kv_heads * n.prefix_tiles;
        int splits = (kBlocks + base - 1) / base;
        n.prefix_splits = splits < 1 ? 1 : splits > most ? most : splits;
    }
    if (own_capacity > 0) {
        n.qo = own_rows <= 16 ? 1 : 2;
        n.own_tiles = (own_rows + 16 * n.qo - 1) / (16 * n.qo);
        const int keys = (own_capacity + kTile - 1) / kTile, most = (keys + 3) / 4;
        const int64_t base = (int64_t)sequences * kv_heads * n.own_tiles;
        const int64_t splits = (kBlocks + base - 1) / base;
        n.own_splits = (int)(splits > most ? most : splits);
    }
    const int slots = n.prefix_splits + n.own_splits;
    n.direct = slots == 1 && n.prefix_splits == 0;
    n.stats_at = aligned_bytes((size_t)slots * n.rows * kCacheWidth * 4);
    n.bytes = n.direct ? 0 : n.stats_at + aligned_bytes((size_t)slots * n.rows * 8);
    return n;
}

template <bool I8>
void launch(const Plan& n, const SharedParams& p, int blocks, hipStream_t s) {
    const dim3 grid(blocks), block(256);
#define RN_SHARED(QP, WP)                                                                   \
    if (n.qo == 1)                                                                          \
        rn_launch(shared_attend_kernel<I8, QP, WP, 1>, grid, block, 0, s, p);               \
    else                                                                                    \
        rn_launch(shared_attend_kernel<I8, QP, WP, 2>, grid, block, 0, s, p)
    if (n.qp == 1) {
        RN_SHARED(1, 1);
    } else if (n.wp == 1) {
        RN_SHARED(2, 1);
    } else if (n.wp == 2) {
        RN_SHARED(2, 2);
    } else {
        RN_SHARED(2, 4);
    }
#undef RN_SHARED
}

int check_shape(int sequences, int queries, int heads, const rn_cache* prefix, int prefix_length, const rn_cache* own,
                int& kv_heads, int& own_capacity) {
    SV_REQUIRE(prefix || own, "neither a prefix nor an own cache");
    SV_REQUIRE(sequences >= 0 && queries >= 0 && heads >= 1, "bad shape");
    SV_REQUIRE(prefix || prefix_length == 0, "prefix_length %d without a prefix", prefix_length);
    kv_heads = own_capacity = 0;
    if (prefix) {
        SV_CHECK(check_cache(prefix, "prefix"));
        SV_REQUIRE(prefix_length >= 0 && prefix_length <= prefix->capacity, "prefix_length must be 0..%d (got %d)",
                   prefix->capacity, prefix_length);
        kv_heads = prefix->kv_heads;
    }
    if (own) {
        SV_CHECK(check_cache(own, "own"));
        SV_REQUIRE(own->sequences >= sequences, "own holds %d sequences, the batch has %d", own->sequences, sequences);
        SV_REQUIRE(!prefix || own->kv_heads == kv_heads, "prefix and own differ in kv_heads");
        kv_heads = own->kv_heads;
        own_capacity = own->capacity;
    }
    SV_REQUIRE(heads % kv_heads == 0 && heads / kv_heads <= 64, "heads (%d) must be 1..64 times kv_heads (%d)", heads,
               kv_heads);
    SV_REQUIRE(sequences <= 65535 && queries <= 65535 &&
                   (int64_t)sequences * queries * heads <= (int64_t)1 << 20,
               "at most 2^20 rows of queries");
    return RN_OK;
}

}  // namespace
}  // namespace rn

using namespace rn;

int rn_attend_shared_workspace(int sequences, int queries, int heads, const rn_cache* prefix, int prefix_length,
                               const rn_cache* own, size_t* bytes) {
    SV_REQUIRE(bytes, "null argument");
    int kv_heads, capacity;
    SV_CHECK(check_shape(sequences, queries, heads, prefix, prefix_length, own, kv_heads, capacity));
    *bytes = 0;
    if (sequences > 0 && queries > 0)
        *bytes = plan_of(sequences, queries, heads, kv_heads, prefix_length, capacity, 0).bytes;
    return RN_OK;
}

int rn_attend_shared(const float* q, int64_t q_stride, float* out, int64_t out_stride, int sequences, int queries,
                     int heads, const rn_cache* prefix, int prefix_length, const rn_cache* own,
                     const int32_t* lengths, const int32_t* counts, float scale, int window, void* workspace,
                     size_t workspace_bytes, int32_t* error, void* stream) {
    int kv_heads, capacity;
    SV_CHECK(check_shape(sequences, queries, heads, prefix, prefix_length, own, kv_heads, capacity));
    SV_REQUIRE(own || !lengths, "lengths without an own cache");
    SV_REQUIRE(scale > 0.0f && scale < INFINITY, "scale must be positive and finite");
    SV_REQUIRE(window >= 0, "window must not be negative (got %d)", window);
    if (window > (1 << 26)) window = 0;  // wider than any sequence
    if (sequences == 0 || queries == 0) return RN_OK;
    SV_REQUIRE(q && out, "null argument");
    SV_REQUIRE(q_stride >= (int64_t)heads * kCacheWidth && out_stride >= (int64_t)heads * kCacheWidth &&
                   q_stride % 4 == 0 && out_stride % 4 == 0 && q_stride <= ((int64_t)1 << 40) &&
                   out_stride <= ((int64_t)1 << 40),
               "q_stride and out_stride must be multiples of 4 that hold a row of %d floats", heads * kCacheWidth);
    const Plan n = plan_of(sequences, queries, heads, kv_heads, prefix_length, capacity, window);
    const size_t needed = plan_of(sequences, queries, heads, kv_heads, prefix_length, capacity, 0).bytes;
    SV_REQUIRE(workspace_bytes >= needed && (workspace || needed == 0), "the workspace holds %zu bytes of %zu",
               workspace ? workspace_bytes : (size_t)0, needed);
    OnDevice on;
    SV_CHECK(on.enter((hipStream_t)stream));
    SV_CHECK(on.pointer(q, 16, "q"));
    SV_CHECK(on.pointer(out, 16, "out"));
    if (prefix_length > 0) SV_CHECK(check_cache_pointers(on, prefix));
    if (own) SV_CHECK(check_cache_pointers(on, own));
    SV_CHECK(on.optional(lengths, 4, "lengths"));
    SV_CHECK(on.optional(counts, 4, "counts"));
    SV_CHECK(on.optional(error, 4, "error"));
    if (!n.direct) SV_CHECK(on.pointer(workspace, 256, "workspace"));

    SharedParams p{};
    p.q = q;
    p.out = out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    if (prefix_length > 0) p.prefix = cache_dev(prefix);
    if (own) p.own = cache_dev(own);
    p.lengths = lengths;
    p.counts = counts;
    p.parts = n.direct ? nullptr : (float*)workspace;
    p.stats = n.direct ? nullptr : (float2*)((char*)workspace + n.stats_at);
    p.error = error;
    p.sequences = sequences;
    p.queries = queries;
    p.kv_heads = kv_heads;
    p.group = heads / kv_heads;
    p.rows = n.rows;
    p.prefix_first = n.prefix_first;
    p.prefix_length = prefix_length;
    p.window = window;
    p.prefix_tiles = n.prefix_tiles;
    p.prefix_splits = n.prefix_splits;
    p.own_tiles = n.own_tiles;
    p.own_splits = n.own_splits;
    p.scale2 = scale * 1.44269504088896340736f;
    const int64_t shared = (int64_t)kv_heads * n.prefix_tiles * n.prefix_splits;
    const int64_t single = (int64_t)sequences * kv_heads * n.own_tiles * n.own_splits;
    hipStream_t s = (hipStream_t)stream;
    const bool mixed = prefix_length > 0 && own && prefix->format != own->format;
    // one launch for both kinds of blocks, or one each where the caches' formats differ
    if (prefix_length > 0) {
        p.prefix_tasks = (int)shared;
        const int blocks = (int)(mixed ? shared : shared + single);
        prefix->format == RN_CACHE_I8 ? launch<true>(n, p, blocks, s) : launch<false>(n, p, blocks, s);
        SV_HIP(hipGetLastError());
    }
    if (own && (mixed || prefix_length == 0)) {
        p.prefix_tasks = 0;
        own->format == RN_CACHE_I8 ? launch<true>(n, p, (int)single, s) : launch<false>(n, p, (int)single, s);
        SV_HIP(hipGetLastError());
    }
    if (!n.direct) {
        rn_launch(shared_join_kernel, dim3((n.rows + 3) / 4), dim3(256), 0, s, p);
        SV_HIP(hipGetLastError());
    }
    return RN_OK;
}
