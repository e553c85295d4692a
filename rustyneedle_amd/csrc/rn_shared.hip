// rn_shared.hip — attention of a batch over one shared prefix and each sequence's
// own cache (rn_attend_shared).
//
// For a query q of a (sequence, token, head), with c = scale log2(e):
//     s_k = q . k_k,  w_k = 2^(c s_k - m),  out = sum w_k v_k / sum w_k,
// over the positions the query sees; any m gives the same value, and the running
// maximum of c s_k keeps every w_k in range. The keys are split over blocks; each
// block leaves (m, sum w_k, sum w_k v_k) of its share, and one more launch joins the
// shares, each times 2^(m - max m). (Small problems: one launch, see plan_of.)
//
// The rows of a block are queries: of every sequence for a share of the prefix (so
// the prefix is read once for all), of one sequence for a share of its own cache.
// v_mfma_f32_32x32x16_f16 (16x16x32 for at most 16 rows) computes scores with keys as
// rows and queries as columns, so a lane holds scores of one query, and they are the
// second product's B operand (keys x queries, against values transposed by
// ds_read_b64_tr_b16) as they are: its k slots may name the keys in any order as long
// as both operands agree.
//
// Precision: int8 codes and fp16 keys are exact in fp16. A query is scaled by a power
// of two (exact) to a peak in [2^13, 2^14) and enters as two fp16 numbers, hi + lo =
// 22 bits; a weight, times 2^14, likewise. Each product is so twice the matrix
// instructions of a single fp16 one, with f32 sums: about 1e-6 from the exact value
// where a single one is off by 2e-4. A value row's scale enters the weight's exponent.
//
// What bounds it (MI355X, traced): 256 8-bit rows over a prefix of 32768 positions on 8
// heads and 256 own caches of 550 keys: 75 us and 5 for the join, where own caches alone
// take 33 us (4.6 TB/s of 4.9) and the prefix 61 (34 GFLOP as fp16 pairs). The vector
// units issue 54% of that time and the matrix units are busy 23%, and the two overlap
// only in part: a round of 32 keys and 32 rows a wave is 16 matrix instructions and about
// 165 others (scales 48, exponentials 32, sums 16, weights as two fp16 numbers 32, the
// maximum, the next tile), 0.8 us a SIMD with two waves and 0.9 with one. fp16 own
// caches of 550 keys: 51 us, 5.6 TB/s.
#include "rn_device.hpp"
#include "rn_serving.hpp"

namespace rn {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

// Weights are held times 2^14 (small ones keep their bits as fp16 pairs), against a
// reference that follows the running maximum once that is 2^1.9 above it: 2^15.9 is
// below the largest fp16 number, and most tiles then rescale nothing.
constexpr int kWeightBits = 14;
constexpr float kSlack = 1.9f, kNoReference = -3e38f;

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
    int prefix_tiles, prefix_splits, prefix_tasks, own_tiles, own_splits, own_tasks;
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

__device__ __forceinline__ float min_of(float a, float b) { return __builtin_fminf(a, b); }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// l 2^d for a sum of weights l, d <= 0. Divided by value scales it may be far from 1
// where the weights are not, so half of d at a time: 2^d alone could be less than the
// smallest float.
__device__ __forceinline__ float scaled_sum(float l, float d) {
    const float half = exp2_of(0.5f * d);
    return l * half * half;
}

// Four int8 codes as fp16: the byte c ^ 0x80 = c + 128 under the exponent of 1024 is
// 1152 + c exactly; less 1152.
__device__ __forceinline__ v2u halves_of_codes(uint32_t codes) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const uint32_t u = codes ^ 0x80808080u;
    const uint32_t a = __builtin_amdgcn_perm(0x64646464u, u, 0x07010700u);
    const uint32_t b = __builtin_amdgcn_perm(0x64646464u, u, 0x07030702u);
    const v2h bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    return v2u{__builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, a) - bias),
               __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, b) - bias)};
}
__device__ __forceinline__ v4u halves_of_codes(uint32_t first, uint32_t second) {
    const v2u a = halves_of_codes(first), b = halves_of_codes(second);
    return v4u{a[0], a[1], b[0], b[1]};
}

// Where the 16-byte chunk `chunk` (0..7) of key row `row` lies in a staged tile:
// rows are 128 bytes, the chunks of eight rows in a row permuted so that the sixteen
// lanes that read one chunk of sixteen rows meet different banks.
__device__ __forceinline__ int staged(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// -1 in a register the compiler cannot see into: with the literal it would turn the fma
// below into a conversion and a subtraction.
__device__ __forceinline__ float opaque_minus_one() {
    float z;
    asm("v_mov_b32 %0, -1.0" : "=v"(z));
    return z;
}

// Both fp16 parts of two numbers, cut towards zero: hi + lo = 20 to 22 bits of each. Four
// instructions (v_fma_mix_f32 takes the half as it is).
__device__ __forceinline__ void split_pair(float a, float b, float minus, uint32_t& hi, uint32_t& lo) {
    typedef __fp16 v2f __attribute__((ext_vector_type(2)));
    const v2f h = __builtin_amdgcn_cvt_pkrtz(a, b);
    const v2f l = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)h[0], minus, a), __builtin_fmaf((float)h[1], minus, b));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

union Frag {
    uint32_t w[4];
    v4u q;
    v8h h;
};

// fp16 values with infinities and NaN among them, where a weight of 0 must not meet
// them: the finite ones, and 1 where a value is +infinity or NaN, -infinity or NaN.
struct OddFrag {
    Frag finite, up, down;
};
__device__ __forceinline__ OddFrag odd_parts(const Frag& a) {
    OddFrag o;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        uint32_t odd = 0, up = 0, down = 0;
#pragma unroll
        for (int h = 0; h < 32; h += 16) {
            const uint32_t v = a.w[x] >> h & 0xffffu, size = v & 0x7fffu;
            if (size >= 0x7c00u) odd |= 0xffffu << h;
            if (size > 0x7c00u || v == 0x7c00u) up |= 0x3c00u << h;
            if (size > 0x7c00u || v == 0xfc00u) down |= 0x3c00u << h;
        }
        o.finite.w[x] = a.w[x] & ~odd;
        o.up.w[x] = up;
        o.down.w[x] = down;
    }
    return o;
}
__device__ __forceinline__ bool any_odd(const Frag& a) {
    uint32_t found = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) found |= (a.w[x] & 0x7c007c00u) + 0x04000400u;  // bit 15 of a half: its exponent is full
    return (found & 0x80008000u) != 0;
}
// What counts of odd values seen, of either sign, add to a sum.
__device__ __forceinline__ float odd_sum(float up, float down) {
    return (up > 0.0f ? __builtin_inff() : 0.0f) - (down > 0.0f ? __builtin_inff() : 0.0f);
}

// The largest of a wave's numbers.
__device__ __forceinline__ int wave_max_i(int v) {
    v = max(v, dpp_move<0xb1>(v));
    v = max(v, dpp_move<0x4e>(v));
    v = max(v, dpp_move<0x141>(v));
    v = max(v, dpp_move<0x140>(v));
    return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
               max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

__device__ __forceinline__ v4f mfma(const Frag& a, const Frag& b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
}

// n / d for 0 <= n < 2^21, 0 < d: the quotient in f32 is off by less than one.
__device__ __forceinline__ int quotient(int n, int d) {
    int q = (int)((float)n * __builtin_amdgcn_rcpf((float)d));
    const int r = n - q * d;
    q -= r < 0;
    return q + (r >= d);
}

// A number that all lanes have: where it was computed by vector instructions the
// compiler otherwise keeps it, and every address made of it, in each lane.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// A row of queries as a lane holds it.
struct Row {
    int lo, hi;  // the local positions it sees
    int id;      // row number in out and the partials, -1: none
    float rs;    // c over the query's scaling
    float mr;    // the reference (log2)
    float l;     // this lane's share of the sum of weights
};

// Which keys a block takes, and of whose rows.
struct Share {
    bool all;            // the rows are every sequence's, not only one's
    int sequence, head, tile;  // tile: which of the rows
    int origin;          // the position of the cache's first key
    int first, last;     // the keys come from [first, last)
    int t0, t1;          // tiles of them
    int slot;            // where the sums go
    const char *keys, *values;
    const float *key_scales, *value_scales;
};

template <bool I8, class Of>
__device__ __forceinline__ Share share_of(const SharedParams& p, bool prefix, bool all, int sequence, int head, int tile,
                                          int split, int splits, int slot) {
    const CacheDev& cache = prefix ? p.prefix : p.own;
    Share s;
    s.all = all;
    s.sequence = sequence;
    s.head = head;
    s.tile = tile;
    s.slot = slot;
    s.origin = prefix ? 0 : p.prefix_length;
    if (all) {
        s.first = p.prefix_first;
        s.last = p.prefix_length;
    } else {
        // from the first position that the tile's first query sees to its last one's own
        const Sequence q = sequence_of(p, sequence);
        int t0 = 0, t1 = q.count;
        if (p.own_tiles > 1) {
            t0 = quotient(tile * Of::kRows, p.group);
            t1 = min(t1, quotient(tile * Of::kRows + Of::kRows - 1, p.group) + 1);
        }
        const int before = p.prefix_length + q.length - q.count - s.origin;
        s.last = uniform(t1 > t0 ? max(min(before + t1, prefix ? p.prefix_length : q.length), 0) : 0);
        s.first = uniform(p.window > 0 ? max(min(before + t0 + 1 - p.window, s.last), 0) : 0);
    }
    // (at most 2^19 tiles times 4096 shares)
    const uint32_t tiles = (uint32_t)(s.last - s.first + Of::kKeys - 1) / Of::kKeys;
    s.t0 = uniform((int)(tiles * (uint32_t)split / (uint32_t)splits));
    s.t1 = uniform((int)(tiles * (uint32_t)(split + 1) / (uint32_t)splits));
    const int64_t base = (prefix ? 0 : (int64_t)sequence * cache.sequence_rows) + (int64_t)head * cache.head_rows;
    s.keys = cache.keys + base * (I8 ? 64 : 128);
    s.values = cache.values + base * (I8 ? 64 : 128);
    s.key_scales = I8 ? cache.key_scales + base : nullptr;
    s.value_scales = I8 ? cache.value_scales + base : nullptr;
    return s;
}

template <bool I8, class Of>
__device__ __forceinline__ Share own_share(const SharedParams& p, int sequence, int head, int tile, int split) {
    return share_of<I8, Of>(p, false, false, sequence, head, tile, split, p.own_splits, p.prefix_splits + split);
}

// Row number r of the block's rows: where its query lies (null: there is none). What
// its sequence's numbers say of it comes after the query has been asked for.
__device__ __forceinline__ const float* query_of(const SharedParams& p, const Share& s, int r, int& b, int& t, int& g) {
    const int T = p.queries, G = p.group;
    if (r >= (s.all ? p.sequences : 1) * T * G) return nullptr;
    b = s.all ? quotient(r, T * G) : s.sequence;
    const int in = s.all ? r - b * T * G : r;
    t = quotient(in, G);
    g = in - t * G;
    return p.q + (int64_t)(b * T + t) * p.q_stride + (s.head * G + g) * kCacheWidth;
}
__device__ __forceinline__ void limits_of(const SharedParams& p, const Share& s, bool there, int b, int t, int g, Row& w) {
    w.id = -1;
    w.lo = 0;
    w.hi = 0x7fffffff;
    w.mr = kNoReference;
    w.l = 0.0f;
    if (!there) return;
    const Sequence q = sequence_of(p, b);
    if (t >= q.count) return;
    const int P = p.prefix_length;
    w.id = (b * p.queries + t) * p.kv_heads * p.group + s.head * p.group + g;
    const int end = P + q.length - q.count + t + 1;
    const int begin = p.window > 0 ? max(end - p.window, 0) : 0;
    w.hi = end - s.origin;
    w.lo = begin - s.origin;
}

// The limits of a row on the prefix as those on its own cache.
__device__ __forceinline__ void own_limits(const SharedParams& p, Row& w) {
    if (w.id < 0) return;
    w.lo -= p.prefix_length;
    w.hi -= p.prefix_length;
}

// A query as two fp16 parts: the lane's values d = STEP s + EACH part + j (j < 8) of
// the DEEP steps s, scaled by a power of two to a peak in [2^13, 2^14).
template <int DEEP, int STEP, int EACH>
__device__ __forceinline__ void query_frags(const SharedParams& p, const Share& share, int r, int part, float minus, Row& w,
                                            Frag (&hi)[DEEP], Frag (&lo)[DEEP]) {
    int b = 0, t = 0, g = 0;
    const float* q = query_of(p, share, r, b, t, g);
    float v[DEEP][8];
#pragma unroll
    for (int s = 0; s < DEEP; ++s) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[s][j] = 0.0f;
        if (q) load_floats<8>(q + STEP * s + EACH * part, v[s]);
    }
    limits_of(p, share, q != nullptr, b, t, g, w);
    float peak = 0.0f;
#pragma unroll
    for (int s = 0; s < DEEP; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) peak = max_of(peak, fabsf(v[s][j]));
    if constexpr (DEEP == 2) peak = max_of(peak, lane_xor<16>(peak));
    peak = max_of(peak, lane_xor<32>(peak));
    const int e = peak < __builtin_inff() ? (int)(__float_as_uint(peak) >> 23) - 127 : 0;
    w.rs = max_of(__builtin_ldexpf(p.scale2, e - 13), 0x1p-126f);
#pragma unroll
    for (int s = 0; s < DEEP; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            split_pair(__builtin_ldexpf(v[s][2 * j], 13 - e), __builtin_ldexpf(v[s][2 * j + 1], 13 - e), minus, hi[s].w[j],
                       lo[s].w[j]);
}

// The least and most of the wave's limits (each lane's over its rows).
__device__ __forceinline__ void wave_limits(int& lo_most, int& hi_least) {
    lo_most = wave_max_i(lo_most);
    hi_least = -wave_max_i(-hi_least);
}

// A value row's scale v enters the exponent, w = 2^(c s + log2 v - m), and is divided out
// again where the weights are summed, so the weights of a row of queries are in range
// whatever scales the keys have that it does not see. Scales below 2^-100 count as 0:
// their codes are cleared, for a scale that is 2^-100 to the sums of weights. Negative
// and infinite ones and NaN give NaN to whom sees them.
constexpr float kLeastScale = 0x1p-100f;
__device__ __forceinline__ float log_scale(float v) {
    const float x = max_of(v, kLeastScale);  // (of a NaN: the least)
    return v >= 0.0f && v < __builtin_inff() ? __builtin_amdgcn_logf(x) : __builtin_nanf("");
}
__device__ __forceinline__ float inverse_scale(float v) {
    const float x = max_of(v, kLeastScale);
    return x < __builtin_inff() ? __builtin_amdgcn_rcpf(x) : 1.0f;
}

// A finished quarter of a row: partial sums, or the output where they are the only ones.
__device__ __forceinline__ void leave(const SharedParams& p, int id, int at, v4f o, float mr, float l, int slot) {
    if (p.parts) {
        const int64_t r = (int64_t)slot * p.rows + id;
        if (at == 0) p.stats[r] = make_float2(mr, l);
        if (l != 0.0f) *reinterpret_cast<v4f*>(p.parts + r * kCacheWidth + at) = o;
    } else {
        const int heads = p.kv_heads * p.group, token = quotient(id, heads);
        *reinterpret_cast<v4f*>(p.out + token * p.out_stride + (id - token * heads) * kCacheWidth + at) =
            l != 0.0f ? o / l : v4f{0, 0, 0, 0};
    }
}

// Joins sums that lie in LDS, [columns][64] and (reference, sum, row) of each: KS x JS of
// them make a row, at columns row_column + k KSTEP + j.
template <int KS, int KSTEP, int JS>
__device__ __forceinline__ void join_columns(const SharedParams& p, const float* sums, const float4* heads, int column,
                                             int part, int slot) {
    float m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < JS; ++j) {
            const float4 h = heads[column + k * KSTEP + j];
            if (h.y != 0.0f) m = max_of(m, h.x);
        }
    const int id = __float_as_int(heads[column].z);
    if (id < 0) return;
    v4f o = v4f{0, 0, 0, 0};
    float l = 0.0f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int j = 0; j < JS; ++j) {
            const int c = column + k * KSTEP + j;
            const float4 h = heads[c];
            const float a = h.y != 0.0f ? exp2_of(h.x - m) : 0.0f;
            const v4f v = *reinterpret_cast<const v4f*>(sums + c * kCacheWidth + ((part ^ (c & 15)) << 2));
            if (h.y != 0.0f) {
                l += scaled_sum(h.y, h.x - m);
                o += a * v;
            }
        }
    leave(p, id, part * 4, o, l != 0.0f ? m : 0.0f, l, slot);
}

// Puts a lane's column of sums (rows d = 16 x + 4 quad + j of it) where join_columns reads it.
__device__ __forceinline__ void put_column(float* sums, float4* heads, int column, int quad, const v4f (&acc)[4],
                                           const Row& w) {
#pragma unroll
    for (int d = 0; d < 4; ++d)
        *reinterpret_cast<v4f*>(sums + column * kCacheWidth + (((d * 4 + quad) ^ (column & 15)) << 2)) = acc[d];
    if (quad == 0) heads[column] = make_float4(w.mr, w.l, __int_as_float(w.id), 0.0f);
}

// The sum of weights over the four lanes of a column.
__device__ __forceinline__ void close_row(Row& w) {
    w.l += lane_xor<16>(w.l);
    w.l += lane_xor<32>(w.l);
}

// Tiles of 32 keys on their way through LDS, for a block of four waves: WM of them hold
// different rows and share each tile, the 4 / WM groups take tiles in turn. Waves of a
// group of one stage for themselves, without barriers. A tile lies in LDS as fp16, with
// its scales, while the next one is put beside it: one barrier a round.
template <bool I8, int WM>
struct Stage {
    static constexpr int kKeys = 32;
    static constexpr int kGroups = 4 / WM, kThreads = 64 * WM;
    static constexpr int kRowBytes = I8 ? 64 : 128, kRowChunks = kRowBytes / 16;
    static constexpr int kTileChunks = kRowChunks * kKeys;      // 16-byte loads a tile of keys, or of values
    static constexpr int kChunks = 2 * kTileChunks / kThreads;  // and a thread, of both
    static constexpr int kTileBytes = kKeys * 128;
    // two tiles of keys, two of values, and two each of key scales, log2 and inverse of value scales
    static constexpr int kScales = 4 * kTileBytes, kGroupBytes = kScales + (I8 ? 6 * kKeys * 4 : 0);

    Share share;
    const int lane, wave, wm, wk, thread;
    char* const stage;

    __device__ __forceinline__ Stage(const Share& s_, char* lds)
        : share(s_), lane(threadIdx.x % 64), wave(__builtin_amdgcn_readfirstlane(threadIdx.x / 64)), wm(wave % WM),
          wk(wave / WM), thread(threadIdx.x % kThreads), stage(lds + wk * kGroupBytes) {}
    __device__ __forceinline__ char* keys_at(int odd) const { return stage + odd * kTileBytes; }
    __device__ __forceinline__ char* values_at(int odd) const { return stage + (2 + odd) * kTileBytes; }
    // which: 0 key scales, 1 log2 and 2 inverse of value scales
    __device__ __forceinline__ float* scales_at(int which, int odd) const {
        return reinterpret_cast<float*>(stage + kScales) + (2 * which + odd) * kKeys;
    }
    __device__ __forceinline__ void sync() const {
        if constexpr (WM == 1)
            wave_lds_sync();
        else
            lds_barrier();
    }

    // This group's tile number n. Past the share its keys are hidden.
    __device__ __forceinline__ int first_key(int n) const { return share.first + (share.t0 + n * kGroups + wk) * kKeys; }
    __device__ __forceinline__ int rounds() const { return (share.t1 - share.t0 + kGroups - 1) / kGroups; }
    __device__ __forceinline__ int end() const { return min(share.last, share.first + share.t1 * kKeys); }

    // Tile m on its way.
    struct Fetched {
        v4u v[kChunks];
        float scale, row[kChunks];
    };
    // Whether chunk number x of this thread is one of values (the same in a whole wave).
    __device__ __forceinline__ bool of_values(int x) const {
        return kChunks > 1 ? x >= kChunks / 2 : wave * 64 >= kTileChunks;
    }
    __device__ __forceinline__ void fetch(int m, Fetched& f) const {
        const int k0 = first_key(m);
        const bool inside = k0 + kKeys <= share.last;  // else key by key
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
            const bool values = of_values(x);
            const int chunk = (thread + x * kThreads) % kTileChunks, r = chunk / kRowChunks, part = chunk % kRowChunks;
            const char* from = values ? share.values : share.keys;
            if (inside) {
                const char* tile = from + (int64_t)k0 * kRowBytes;
                f.v[x] = *reinterpret_cast<const v4u*>(tile + (uint32_t)(r * kRowBytes + part * 16));
                if (I8 && values) {
                    const char* scales = reinterpret_cast<const char*>(share.value_scales + k0);
                    f.row[x] = *reinterpret_cast<const float*>(scales + (uint32_t)(r * 4));
                }
            } else {
                const int key = min(k0 + r, share.last - 1);
                f.v[x] = *reinterpret_cast<const v4u*>(from + (int64_t)key * kRowBytes + part * 16);
                if (I8 && values) f.row[x] = share.value_scales[key];
            }
        }
        if (I8 && wm == 0) {  // the halves of the group's first wave take a scale each
            const bool values = lane >= kKeys;
            int key = k0 + lane % kKeys;
            if (!inside) key = min(key, share.last - 1);
            f.scale = (values ? share.value_scales : share.key_scales)[key];
        }
    }
    // ODD: whether m is.
    template <int ODD>
    __device__ __forceinline__ void put(int m, const Fetched& f) const {
#pragma unroll
        for (int x = 0; x < kChunks; ++x) {
            const bool values = of_values(x);
            const int chunk = (thread + x * kThreads) % kTileChunks, r = chunk / kRowChunks, part = chunk % kRowChunks;
            char* to = values ? values_at(ODD) : keys_at(ODD);
            v4u v = f.v[x];
            if constexpr (I8) {
                if (values && f.row[x] < kLeastScale) v = v4u{0, 0, 0, 0};
                *reinterpret_cast<v4u*>(to + staged(r, 2 * part)) = halves_of_codes(v[0], v[1]);
                *reinterpret_cast<v4u*>(to + staged(r, 2 * part + 1)) = halves_of_codes(v[2], v[3]);
            } else {
                // values past the last hold zeros: a weight of 0 must not meet a NaN
                if (values && first_key(m) + r >= share.last) v = v4u{0, 0, 0, 0};
                *reinterpret_cast<v4u*>(to + staged(r, part)) = v;
            }
        }
        if (I8 && wm == 0) {
            // (of hidden keys past the last, which are the last one's again, the inverse is finite)
            if (lane < kKeys) {
                scales_at(0, ODD)[lane] = f.scale;
            } else {
                scales_at(1, ODD)[lane - kKeys] = log_scale(f.scale);
                scales_at(2, ODD)[lane - kKeys] = inverse_scale(f.scale);
            }
        }
    }
};

// A share of the keys for ROWS query rows a wave, ROWS WM a block. For a score tile of
// keys x queries a lane (query, part) holds the scores of 4 keys out of every
// 4 kParts, and those are its operand of the second product:
//   ROWS 16: v_mfma_f32_16x16x32_f16, two tiles of 16 keys, 4 parts;
//   ROWS 32: v_mfma_f32_32x32x16_f16, one of 32 keys, 2 parts.
// The vector unit issues nothing for about 9 cycles at each matrix instruction, and the
// larger ones are half as many: a round of 32 rows, 32 keys takes 900 cycles with them
// against 1300 with two tiles of the smaller (both with everything else at hand).
template <bool I8, int ROWS, int WM>
struct Job {
    typedef Stage<I8, WM> S;
    typedef typename S::Fetched Fetched;
    typedef float vacc __attribute__((ext_vector_type(ROWS == 32 ? 16 : 4)));
    static constexpr int kKeys = S::kKeys, kGroups = S::kGroups, kRows = ROWS * WM, kParts = 64 / ROWS;
    static constexpr int kScores = kKeys / kParts;                // of a lane and tile: 8 or 16
    static constexpr int kTiles = ROWS == 32 ? 1 : 2;             // score tiles a tile of keys
    static constexpr int kDeep = ROWS == 32 ? 4 : 2;              // steps over d of a score
    static constexpr int kSteps = ROWS == 32 ? 2 : 1;             // steps over the keys of a product
    static constexpr int kWide = ROWS == 32 ? 2 : 4;              // tiles of d of a product
    static constexpr int kColumns = 4 * ROWS;
    static constexpr int kJoinBytes = kGroups > 1 ? kColumns * (kCacheWidth * 4 + 16) : 0;
    static constexpr int kLds = kGroups * S::kGroupBytes > kJoinBytes ? kGroups * S::kGroupBytes : kJoinBytes;

    const SharedParams& p;
    S st;
    char* const lds;
    const int col, part;
    Row row;
    Frag qh[kDeep], ql[kDeep];
    vacc acc[kWide];
    int end, lo_most, hi_least;
    float minus;

    __device__ __forceinline__ Job(const SharedParams& p_, const Share& s_, char* lds_)
        : p(p_), st(s_, lds_), lds(lds_), col(st.lane % ROWS), part(st.lane / ROWS) {}

    __device__ __forceinline__ static vacc multiply(const Frag& a, const Frag& b, vacc c) {
        if constexpr (ROWS == 32)
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(a.h, b.h, c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.h, b.h, c, 0, 0, 0);
    }
    // Where a lane's scores 4 x .. 4 x + 3 stand in the tile.
    __device__ __forceinline__ int key_of(int x) const { return x * 4 * kParts + part * 4; }
    __device__ __forceinline__ bool hidden(int key) const { return key < row.lo || key >= row.hi || key >= end; }

    __device__ __forceinline__ void read_scales(int which, int odd, float (&v)[kScores]) const {
#pragma unroll
        for (int x = 0; x < kScores / 4; ++x) {
            const v4f t = *reinterpret_cast<const v4f*>(st.scales_at(which, odd) + key_of(x));
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * x + j] = t[j];
        }
    }
    __device__ __forceinline__ void read_keys(int odd, Frag (&k)[kTiles][kDeep]) const {
#pragma unroll
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
            for (int d = 0; d < kDeep; ++d)
                k[x][d].q = *reinterpret_cast<const v4u*>(st.keys_at(odd) + staged(x * 16 + col, d * kParts + part));
    }
    // The values of a step over the keys and a tile of d, keys in the order of the weights.
    __device__ __forceinline__ Frag values_frag(int odd, int step, int d) const {
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        const int sixteen = st.lane / 16 % (ROWS / 16), l = st.lane % 16;  // which sixteen d of the tile
        Frag a;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = step * 16 + x * 4 * kParts + part * 4 + l / 4;
            const char* at = st.values_at(odd) + staged(r, (d * (ROWS / 16) + sixteen) * 2 + l % 4 / 2) + l % 2 * 8;
            const v2u two = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
            a.w[2 * x] = two[0];
            a.w[2 * x + 1] = two[1];
        }
        return a;
    }
    // The scores of a tile over scale: keys as rows, queries as columns.
    __device__ __forceinline__ void scores(const Frag (&k)[kTiles][kDeep], vacc (&c)[kTiles]) const {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
#pragma unroll
            for (int x = 0; x < kTiles; ++x) c[x] = multiply(k[x][d], ql[d], d == 0 ? vacc{} : c[x]);
#pragma unroll
            for (int x = 0; x < kTiles; ++x) c[x] = multiply(k[x][d], qh[d], c[x]);
        }
    }
    __device__ __forceinline__ static void unpack(const vacc (&c)[kTiles], float (&s)[kScores]) {
#pragma unroll
        for (int x = 0; x < kTiles; ++x)
#pragma unroll
            for (int j = 0; j < kScores / kTiles; ++j) s[x * (kScores / kTiles) + j] = c[x][j];
    }

    // One round: tile n; what was fetched is put down, and more asked for. ODD: whether
    // n is.
    template <int ODD>
    __device__ __forceinline__ void turn(int n, Fetched& f) {
        st.sync();  // tile n - 1 is done with, tile n is there
        Frag k[kTiles][kDeep];
        read_keys(ODD, k);
        vacc raw[kTiles];
        scores(k, raw);
        float s[kScores];
        unpack(raw, s);
        if constexpr (I8) {
            float scale[kScores], logs[kScores];
            read_scales(0, ODD, scale);
            read_scales(1, ODD, logs);
#pragma unroll
            for (int j = 0; j < kScores; ++j) s[j] = __builtin_fmaf(s[j] * scale[j], row.rs, logs[j]);
        }
        const int k0 = st.first_key(n);
        bool odd = false;  // fp16 values that are not finite, where some row does not see them
        if (lo_most > k0 || hi_least < k0 + kKeys) {
#pragma unroll
            for (int j = 0; j < kScores; ++j)
                if (hidden(k0 + key_of(j / 4) + j % 4)) s[j] = -__builtin_inff();
            if constexpr (!I8) {
#pragma unroll
                for (int x = 0; x < kSteps; ++x)
#pragma unroll
                    for (int d = 0; d < kWide; ++d) odd |= any_odd(values_frag(ODD, x, d));
                odd = __any(odd);
            }
        }
        // ---- the reference: looked at across the lanes of a column only where one has to move
        float m = max_of(s[0], s[1]);
#pragma unroll
        for (int j = 2; j < kScores; j += 2) m = max_of(max_of(m, s[j]), s[j + 1]);
        if constexpr (!I8) m *= row.rs;
        if (__any(m > row.mr + kSlack)) {
            float y = max_of(m, lane_xor<32>(m));
            if constexpr (kParts == 4) y = max_of(y, lane_xor<16>(y));
            // (a column by its own scores alone: the others of the tile do not matter to it)
            y = y > row.mr + kSlack ? y : row.mr;
            const float alpha = exp2_of(row.mr - y);
            row.l = scaled_sum(row.l, row.mr - y);
#pragma unroll
            for (int d = 0; d < kWide; ++d) acc[d] *= alpha;
            row.mr = y;
        }
        // ---- weights
        const float c = (float)kWeightBits - row.mr;
        float inverse[kScores];
        if constexpr (I8) read_scales(2, ODD, inverse);
        Frag hi[kSteps], lo[kSteps];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < kScores; j += 2) {
            float w[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (I8) {
                    w[x] = exp2_of(s[j + x] + c);
                    sum[x] = __builtin_fmaf(w[x], inverse[j + x], sum[x]);
                } else {
                    w[x] = exp2_of(__builtin_fmaf(s[j + x], row.rs, c));
                    sum[x] += w[x];
                }
            }
            split_pair(w[0], w[1], minus, hi[j / 8].w[j % 8 / 2], lo[j / 8].w[j % 8 / 2]);
        }
        row.l += sum[0] + sum[1];
        // ---- values
        if (odd) {
            odd_products<ODD>(k0, hi, lo);
        } else {
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
                Frag a[kWide];
#pragma unroll
                for (int d = 0; d < kWide; ++d) a[d] = values_frag(ODD, x, d);
#pragma unroll
                for (int d = 0; d < kWide; ++d) acc[d] = multiply(a[d], lo[x], acc[d]);
#pragma unroll
                for (int d = 0; d < kWide; ++d) acc[d] = multiply(a[d], hi[x], acc[d]);
            }
        }
        st.template put<1 - ODD>(n + 1, f);
        st.fetch(n + 2, f);
    }

    // The products with a tile of fp16 values that holds infinities or NaN: those reach
    // the rows that see their keys, as counts.
    template <int ODD>
    __device__ __forceinline__ void odd_products(int k0, const Frag (&hi)[kSteps], const Frag (&lo)[kSteps]) {
        Frag seen[kSteps];
#pragma unroll
        for (int j = 0; j < kScores; j += 2)
            seen[j / 8].w[j % 8 / 2] = (hidden(k0 + key_of(j / 4) + j % 4) ? 0u : 0x3c00u) |
                                       (hidden(k0 + key_of(j / 4) + j % 4 + 1) ? 0u : 0x3c000000u);
#pragma unroll
        for (int d = 0; d < kWide; ++d) {
            vacc up{}, down{};
#pragma unroll
            for (int x = 0; x < kSteps; ++x) {
                const OddFrag o = odd_parts(values_frag(ODD, x, d));
                acc[d] = multiply(o.finite, lo[x], acc[d]);
                acc[d] = multiply(o.finite, hi[x], acc[d]);
                up = multiply(o.up, seen[x], up);
                down = multiply(o.down, seen[x], down);
            }
#pragma unroll
            for (int y = 0; y < kCacheWidth / kWide / kParts; ++y) acc[d][y] += odd_sum(up[y], down[y]);
        }
    }

    // The tiles of the share; f: the first one, on its way.
    __device__ __forceinline__ void pass(Fetched& f) {
        if (st.share.t0 >= st.share.t1) return;
        end = st.end();
        lo_most = row.lo;
        hi_least = row.hi;
        wave_limits(lo_most, hi_least);
        hi_least = min(hi_least, end);
        st.template put<0>(0, f);
        st.fetch(1, f);
        const int rounds = st.rounds();
        for (int n = 0; n < rounds; n += 2) {
            turn<0>(n, f);
            if (n + 1 < rounds) turn<1>(n + 1, f);
        }
    }

    // BOTH: the share is of the prefix, and the sequence's own keys follow.
    template <bool BOTH>
    __device__ __forceinline__ void run() {
        Fetched f;
        if (st.share.t0 < st.share.t1) st.fetch(0, f);  // on its way while the queries are split
        minus = opaque_minus_one();
        query_frags<kDeep, 8 * kParts, 8>(p, st.share, st.share.tile * kRows + st.wm * ROWS + col, part, minus, row, qh, ql);
#pragma unroll
        for (int d = 0; d < kWide; ++d) acc[d] = vacc{};
        pass(f);
        if constexpr (BOTH) {
            st.share = own_share<I8, Job>(p, st.share.sequence, st.share.head, st.share.tile, 0);
            if (st.share.t0 < st.share.t1) st.fetch(0, f);
            own_limits(p, row);
            st.sync();
            pass(f);
        }
        if constexpr (kParts == 4) row.l += lane_xor<16>(row.l);
        row.l += lane_xor<32>(row.l);
        // a lane's sums: of d = ROWS x + 4 kParts y + 4 part + j
        constexpr int kRuns = kCacheWidth / kWide / kParts / 4;
        if constexpr (kGroups == 1) {
            if (row.id >= 0) {
#pragma unroll
                for (int d = 0; d < kWide; ++d)
#pragma unroll
                    for (int y = 0; y < kRuns; ++y)
                        leave(p, row.id, d * ROWS + y * 4 * kParts + part * 4,
                              v4f{acc[d][4 * y], acc[d][4 * y + 1], acc[d][4 * y + 2], acc[d][4 * y + 3]}, row.mr, row.l,
                              st.share.slot);
            }
        } else {
            // every wave's sums go to LDS: [wave][ROWS] columns
            __syncthreads();
            float* sums = reinterpret_cast<float*>(lds);
            float4* heads = reinterpret_cast<float4*>(lds + kColumns * kCacheWidth * 4);
            const int column = st.wave * ROWS + col;
#pragma unroll
            for (int d = 0; d < kWide; ++d)
#pragma unroll
                for (int y = 0; y < kRuns; ++y)
                    *reinterpret_cast<v4f*>(sums + column * kCacheWidth +
                                            (((d * ROWS / 4 + y * kParts + part) ^ (column & 15)) << 2)) =
                        v4f{acc[d][4 * y], acc[d][4 * y + 1], acc[d][4 * y + 2], acc[d][4 * y + 3]};
            if (part == 0) heads[column] = make_float4(row.mr, row.l, __int_as_float(row.id), 0.0f);
            __syncthreads();
            for (int x = threadIdx.x; x < kRows * 16; x += 256)
                join_columns<kGroups, WM * ROWS, 1>(p, sums, heads, x / 16, x % 16, st.share.slot);
        }
    }
};

// The same for at most four rows (fp16: eight), a decode step of one sequence: all
// sixteen columns of a score tile for one query would waste fifteen of its lanes'
// exponentials, so the columns are (row, key tile): every row's query fills four (two),
// the scores of the key tiles of a step are taken from one column each, and each column
// keeps sums of its own, joined at the end. A step is 4 KB of keys and 4 KB of values. Keys go straight from memory into the matrix instructions
// (their values d in the order 16 quad + 8 s + j, so that a lane's are consecutive);
// values lie in LDS as they are in memory and 8-bit ones become fp16 after
// ds_read_b64_tr_b8.
template <bool I8>
struct FewJob {
    static constexpr int kTiles = I8 ? 4 : 2, kKeys = 16 * kTiles, kRows = 16 / kTiles, kKeyLoads = 4, kValueLoads = 4;
    static constexpr int kValueBytes = kKeys * (I8 ? 64 : 128);
    static constexpr int kJoinBytes = 4 * kRows * (kCacheWidth * 4 + 16);
    static constexpr int kLds = 4 * kValueBytes > kJoinBytes ? 4 * kValueBytes : kJoinBytes;

    const SharedParams& p;
    Share share;
    char* const lds;
    const int lane, col, quad, wave, kt;
    char* stage_v;
    Row row;
    Frag qh[2], ql[2];
    v4f acc[4];
    float minus;

    __device__ __forceinline__ FewJob(const SharedParams& p_, const Share& s_, char* lds_)
        : p(p_), share(s_), lds(lds_), lane(threadIdx.x % 64), col(lane % 16), quad(lane / 16), wave(threadIdx.x / 64),
          kt(col % kTiles) {
        stage_v = lds + wave * kValueBytes;
    }

    // 8-bit values: rows of 64 bytes, their 16-byte chunks permuted so that the eight
    // rows a quarter of the wave reads at once lie in different banks.
    __device__ __forceinline__ static int raw(int r, int chunk) {
        return r * 64 + ((chunk ^ ((r >> 1 & 1) | (r >> 4 & 1) << 1)) << 4);
    }

    struct Fetched {
        v4u k[kKeyLoads], v[kValueLoads];
        v4f ks, vs;
    };
    __device__ __forceinline__ void fetch(int t, Fetched& f) const {
        const int k0 = share.first + t * kKeys;
#pragma unroll
        for (int c = 0; c < kKeyLoads; ++c) {
            const int key = min(k0 + (I8 ? c : c / 2) * 16 + col, share.last - 1);
            f.k[c] = *reinterpret_cast<const v4u*>(share.keys + (int64_t)key * (I8 ? 64 : 128) +
                                                     (I8 ? quad * 16 : quad * 32 + c % 2 * 16));
        }
#pragma unroll
        for (int c = 0; c < kValueLoads; ++c) {
            const int chunk = lane + c * 64, key = min(k0 + chunk / (I8 ? 4 : 8), share.last - 1);
            f.v[c] = *reinterpret_cast<const v4u*>(share.values + (int64_t)key * (I8 ? 64 : 128) +
                                                     chunk % (I8 ? 4 : 8) * 16);
        }
        if constexpr (I8) {
            typedef float v4a __attribute__((ext_vector_type(4), aligned(4)));
            const int at = k0 + kt * 16 + quad * 4;
            if (k0 + kKeys <= share.last) {
                f.ks = *reinterpret_cast<const v4a*>(share.key_scales + at);
                f.vs = *reinterpret_cast<const v4a*>(share.value_scales + at);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = min(at + j, share.last - 1);
                    f.ks[j] = share.key_scales[key];
                    f.vs[j] = share.value_scales[key];
                }
            }
        }
    }

    __device__ __forceinline__ bool hidden(int key) const { return key < row.lo || key >= row.hi || key >= share.last; }

    // Whether the fp16 values in f have an infinity or NaN among them.
    __device__ __forceinline__ bool has_odd(const Fetched& f) const {
        if constexpr (I8) return false;
        typedef unsigned short v2s __attribute__((ext_vector_type(2)));
        v2s most = {0, 0};
#pragma unroll
        for (int c = 0; c < kValueLoads; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                most = __builtin_elementwise_max(most, __builtin_bit_cast(v2s, f.v[c][j] & 0x7fff7fffu));
        return __any(most[0] >= 0x7c00 || most[1] >= 0x7c00);
    }

    __device__ __forceinline__ Frag half_frag(int st, int d) const {
        typedef __attribute__((address_space(3))) v4s lds_v4s;
        Frag a;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int r = st * 32 + y * 16 + quad * 4 + col / 4;
            char* at = stage_v + staged(r, d * 2 + col % 4 / 2) + col % 2 * 8;
            const v2u part = __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
            a.w[2 * y] = part[0];
            a.w[2 * y + 1] = part[1];
        }
        return a;
    }

    // The tile in f, whose values go to LDS; `next` is asked for as soon as f is used up.
    template <bool MASKED>
    __device__ __forceinline__ void step(int t, Fetched& f, int next) {
        const int k0 = share.first + t * kKeys, mine = k0 + kt * 16 + quad * 4;  // this lane's four keys
        wave_lds_sync();  // the tile before has been read
        if constexpr (I8) {
            if (__any(min_of(min_of(f.vs[0], f.vs[1]), min_of(f.vs[2], f.vs[3])) < kLeastScale)) {
#pragma unroll 1
                for (int c = 0; c < kValueLoads; ++c) {
                    const float scale = share.value_scales[min(k0 + (lane + c * 64) / 4, share.last - 1)];
#pragma unroll
                    for (int x = 0; x < kValueLoads; ++x)
                        if (x == c && scale < kLeastScale) f.v[x] = v4u{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int c = 0; c < kValueLoads; ++c) {
            const int chunk = lane + c * 64;
            if constexpr (I8) {
                *reinterpret_cast<v4u*>(stage_v + raw(chunk / 4, chunk % 4)) = f.v[c];
            } else {
                const bool in = k0 + chunk / 8 < share.last;
                *reinterpret_cast<v4u*>(stage_v + staged(chunk / 8, chunk % 8)) = in ? f.v[c] : v4u{0, 0, 0, 0};
            }
        }
        // a weight of 0, for another tile's keys too, must not meet an infinity or NaN
        const bool odd = MASKED && has_odd(f);
        // ---- scores: each key tile against every column, one column's kept
        v4f s = v4f{0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < kTiles; ++x) {
            Frag a[2];
            if constexpr (I8) {
                a[0].q = halves_of_codes(f.k[x][0], f.k[x][1]);
                a[1].q = halves_of_codes(f.k[x][2], f.k[x][3]);
            } else {
                a[0].q = f.k[2 * x];
                a[1].q = f.k[2 * x + 1];
            }
            v4f c = v4f{0, 0, 0, 0};
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                c = mfma(a[d], ql[d], c);
                c = mfma(a[d], qh[d], c);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = kt == x ? c[j] : s[j];
        }
        v4f inverse = v4f{1, 1, 1, 1};
        if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[j] = __builtin_fmaf(s[j] * f.ks[j], row.rs, log_scale(f.vs[j]));
                inverse[j] = inverse_scale(f.vs[j]);
            }
        }
        if (next >= 0) fetch(next, f);
        if constexpr (MASKED) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (hidden(mine + j)) s[j] = -__builtin_inff();
        }
        const float m = max_of(max_of(s[0], s[1]), max_of(s[2], s[3])) * (I8 ? 1.0f : row.rs);
        if (__any(m > row.mr + kSlack)) {
            float y = max_of(m, lane_xor<16>(m));
            y = max_of(y, lane_xor<32>(y));
            // (a column by its own scores alone: the others of the tile do not matter to it)
            y = y > row.mr + kSlack ? y : row.mr;
            const float alpha = exp2_of(row.mr - y);
            row.l = scaled_sum(row.l, row.mr - y);
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= alpha;
            row.mr = y;
        }
        const float c = (float)kWeightBits - row.mr;
        float x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = exp2_of(I8 ? s[j] + c : __builtin_fmaf(s[j], row.rs, c));
            row.l = __builtin_fmaf(x[j], inverse[j], row.l);
        }
        uint32_t hi[2], lo[2];
        split_pair(x[0], x[1], minus, hi[0], lo[0]);
        split_pair(x[2], x[3], minus, hi[1], lo[1]);
        wave_lds_sync();
        // ---- values: a column has weights for its own key tile alone
        typedef int v2i __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) v2i lds_v2i;
#pragma unroll
        for (int st = 0; st < kTiles / 2; ++st) {
            Frag wh, wl;
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    wh.w[2 * y + z] = kt == 2 * st + y ? hi[z] : 0u;
                    wl.w[2 * y + z] = kt == 2 * st + y ? lo[z] : 0u;
                }
            if (!I8 && odd) {  // as Job::odd_products
                Frag seen;
#pragma unroll
                for (int z = 0; z < 4; ++z) {
                    const int at = k0 + z / 2 * 16 + quad * 4 + z % 2 * 2;
                    seen.w[z] = kt != z / 2 ? 0u : (hidden(at) ? 0u : 0x3c00u) | (hidden(at + 1) ? 0u : 0x3c000000u);
                }
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    const OddFrag o = odd_parts(half_frag(st, d));
                    acc[d] = mfma(o.finite, wl, acc[d]);
                    acc[d] = mfma(o.finite, wh, acc[d]);
                    const v4f up = mfma(o.up, seen, v4f{0, 0, 0, 0}), down = mfma(o.down, seen, v4f{0, 0, 0, 0});
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[d][j] += odd_sum(up[j], down[j]);
                }
                continue;
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                Frag a;
                if constexpr (I8) {
                    const int y = col / 2, r = st * 32 + y / 4 * 16 + quad * 4 + y % 4;
                    char* at = stage_v + raw(r, d) + col % 2 * 8;
                    const v2i part = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_v2i*)at);
                    a.q = halves_of_codes((uint32_t)part[0], (uint32_t)part[1]);
                } else {
                    a = half_frag(st, d);
                }
                acc[d] = mfma(a, wl, acc[d]);
                acc[d] = mfma(a, wh, acc[d]);
            }
        }
    }

    // The tiles of the share; f: this wave's first one, on its way.
    __device__ __forceinline__ void pass(Fetched& f) {
        int lo_most = row.lo, hi_least = row.hi;
        wave_limits(lo_most, hi_least);
        hi_least = min(hi_least, share.last);
        for (int t = share.t0 + wave; t < share.t1; t += 4) {
            const int k0 = share.first + t * kKeys, next = t + 4 < share.t1 ? t + 4 : -1;
            if (lo_most > k0 || hi_least < k0 + kKeys || has_odd(f))
                step<true>(t, f, next);
            else
                step<false>(t, f, next);
        }
    }

    template <bool BOTH>
    __device__ __forceinline__ void run() {
        Fetched f;
        if (share.t0 + wave < share.t1) fetch(share.t0 + wave, f);
        minus = opaque_minus_one();
        query_frags<2, 8, 16>(p, share, share.tile * kRows + col / kTiles, quad, minus, row, qh, ql);
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[d] = v4f{0, 0, 0, 0};
        pass(f);
        if constexpr (BOTH) {
            share = own_share<I8, FewJob>(p, share.sequence, share.head, share.tile, 0);
            if (share.t0 + wave < share.t1) fetch(share.t0 + wave, f);
            own_limits(p, row);
            pass(f);
        }
        close_row(row);
        join_tiles();
        __syncthreads();
        float* sums = reinterpret_cast<float*>(lds);
        float4* heads = reinterpret_cast<float4*>(lds + 4 * kRows * kCacheWidth * 4);
        if (kt == 0) put_column(sums, heads, wave * kRows + col / kTiles, quad, acc, row);
        __syncthreads();
        // sixteen threads a row, each of four waves' columns of it
        if (threadIdx.x < kRows * 16)
            join_columns<4, kRows, 1>(p, sums, heads, (int)threadIdx.x / 16, threadIdx.x % 16, share.slot);
    }

    template <int CTRL>
    __device__ __forceinline__ static float neighbour(float v) {
        return __int_as_float(dpp_move<CTRL>(__float_as_int(v)));
    }
    // Joins a row's columns, neighbours among the lanes, in all of them. (Left to the one
    // wave that joins the four, sixteen columns a row took it 2.5 us: 16 sequences over
    // 600 positions 11.6 us against 10.5.)
    __device__ __forceinline__ void join_tiles() {
        float m = row.l != 0.0f ? row.mr : -__builtin_inff();
        m = max_of(m, neighbour<0xb1>(m));
        if constexpr (kTiles == 4) m = max_of(m, neighbour<0x4e>(m));
        const float a = exp2_of(row.mr - m);
        const bool some = row.l != 0.0f;
        row.l = some ? scaled_sum(row.l, row.mr - m) : 0.0f;
        row.l += neighbour<0xb1>(row.l);
        if constexpr (kTiles == 4) row.l += neighbour<0x4e>(row.l);
        row.mr = m;
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v = some ? acc[d][j] * a : 0.0f;
                v += neighbour<0xb1>(v);
                if constexpr (kTiles == 4) v += neighbour<0x4e>(v);
                acc[d][j] = v;
            }
    }
};

// A sequence with bad numbers, where no join follows.
__device__ __forceinline__ void refuse(const SharedParams& p, int sequence) {
    if (!sequence_of(p, sequence).bad) return;
    const int width = p.kv_heads * p.group * kCacheWidth;
    for (int i = threadIdx.x; i < p.queries * width; i += 256) {
        const int t = i / width;
        p.out[(int64_t)(sequence * p.queries + t) * p.out_stride + (i - t * width)] = __builtin_nanf("");
    }
    if (p.error && threadIdx.x == 0) *p.error = RN_ERR_ARGUMENT;
}

template <bool I8, int Q, int W>
struct JobOf {
    typedef Job<I8, 16 * Q, W> type;
};
template <bool I8>
struct JobOf<I8, 0, 1> {  // at most four rows
    typedef FewJob<I8> type;
};

template <bool I8, int QP, int WP, int QO>
constexpr int lds_of() {
    typedef typename JobOf<I8, QP, WP>::type Prefix;
    typedef typename JobOf<I8, QO, 1>::type Own;
    return Prefix::kLds > Own::kLds ? Prefix::kLds : Own::kLds;
}

// (the registers of 16-bit tiles allow two)
template <bool I8, int QP, int WP, int QO>
constexpr int blocks_a_cu() {
    return I8 && lds_of<I8, QP, WP, QO>() <= 160 * 1024 / 3 ? 3 : 2;
}

// Prefix tasks are (key head, share, rows) of the prefix, the others (sequence, key
// head, share, rows) of the own caches. A block of the first kind computes and one of
// the second mostly loads; those of the prefix come first, as they take longest (256 rows
// over 32768 positions and 550 of their own: 77 us; dealt out in turn, 95).
template <bool I8, int QP, int WP, int QO>
__global__ __launch_bounds__(256, (blocks_a_cu<I8, QP, WP, QO>())) void shared_attend_kernel(const SharedParams p) {
    typedef typename JobOf<I8, QP, WP>::type Prefix;
    typedef typename JobOf<I8, QO, 1>::type Own;
    __shared__ __attribute__((aligned(16))) char lds[lds_of<I8, QP, WP, QO>()];
    const bool prefix = (int)blockIdx.x < p.prefix_tasks;
    const int rest = prefix ? blockIdx.x : blockIdx.x - p.prefix_tasks;
    if (prefix) {
        const int share = uniform(quotient(rest, p.prefix_tiles)), tile = rest - share * p.prefix_tiles;
        const int head = uniform(quotient(share, p.prefix_splits)), split = share - head * p.prefix_splits;
        Prefix(p, share_of<I8, Prefix>(p, true, true, 0, head, tile, split, p.prefix_splits, split), lds).template run<false>();
    } else {
        const int share = uniform(quotient(rest, p.own_tiles)), tile = rest - share * p.own_tiles;
        const int pair = uniform(quotient(share, p.own_splits)), split = share - pair * p.own_splits;
        const int sequence = uniform(quotient(pair, p.kv_heads)), head = pair - sequence * p.kv_heads;
        Own(p, own_share<I8, Own>(p, sequence, head, tile, split), lds).template run<false>();
        if (!p.parts) refuse(p, sequence);
    }
}

// Where the work is small: every block reads the prefix and the own cache of its rows,
// and nothing is shared or joined.
template <bool I8, int Q>
__global__ __launch_bounds__(256, (blocks_a_cu<I8, Q, 1, Q>())) void alone_attend_kernel(const SharedParams p) {
    typedef typename JobOf<I8, Q, 1>::type Rows;
    __shared__ __attribute__((aligned(16))) char lds[Rows::kLds];
    const int pair = uniform(quotient(blockIdx.x, p.own_tiles)), tile = blockIdx.x - pair * p.own_tiles;
    const int sequence = uniform(quotient(pair, p.kv_heads)), head = pair - sequence * p.kv_heads;
    Rows(p, share_of<I8, Rows>(p, true, false, sequence, head, tile, 0, 1, 0), lds).template run<true>();
    refuse(p, sequence);
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
    const int slots = p.prefix_splits + p.own_splits;
    // (asked for with the sequence's numbers; of rows that do not count they mean nothing)
    float2 st = lane < slots ? p.stats[(int64_t)lane * p.rows + id] : make_float2(0.0f, 0.0f);
    const Sequence s = sequence_of(p, b);
    float* out = p.out + token * p.out_stride + (id - token * heads) * kCacheWidth;
    if (s.bad) {
        out[lane] = __builtin_nanf("");
        if (p.error && lane == 0) *p.error = RN_ERR_ARGUMENT;
        return;
    }
    if (token - b * p.queries >= s.count) return;
    v4f o = v4f{0, 0, 0, 0};
    float l = 0.0f, most = -__builtin_inff();
    for (int k0 = 0; k0 < slots; k0 += 64) {
        if (k0 > 0) st = k0 + lane < slots ? p.stats[(int64_t)(k0 + lane) * p.rows + id] : make_float2(0.0f, 0.0f);
        const float m = max_of(most, wave_max(st.y != 0.0f ? st.x : -__builtin_inff()));
        if (k0 > 0 && m > most) {
            l = scaled_sum(l, most - m);
            o *= exp2_of(most - m);
        }
        most = m;
        const float weight = st.y != 0.0f ? exp2_of(st.x - m) : 0.0f;
        if (st.y != 0.0f) l += scaled_sum(st.y, st.x - m);
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
    // row tiles: 16 qp wp rows of the prefix, 16 qo of an own cache; 0: the few rows of FewJob
    int rows = 0, qp = 0, wp = 1, qo = 0;
    int prefix_first = 0, prefix_tiles = 0, prefix_splits = 0, own_tiles = 0, own_splits = 0;
    size_t stats_at = 0, bytes = 0;
    bool direct = false, alone = false;
};

constexpr int kCus = 256;
constexpr int kRoundKeys = 32;  // keys a group of waves takes at once of the prefix
constexpr int kAloneKeys = 768;  // keys up to which a block reads the prefix and its own cache
constexpr int kOwnKeys = 256;   // keys of an own cache (half of them taken) that cost about a round

int few_rows(const rn_cache* c) { return c->format == RN_CACHE_I8 ? FewJob<true>::kRows : FewJob<false>::kRows; }

Plan plan_of(int sequences, int queries, int heads, const rn_cache* prefix, int prefix_length, const rn_cache* own,
             int window) {
    Plan n;
    const int kv_heads = (prefix ? prefix : own)->kv_heads, own_capacity = own ? own->capacity : 0;
    const int group = heads / kv_heads;
    n.rows = sequences * queries * heads;
    const int shared_rows = sequences * queries * group, own_rows = queries * group;
    // A short prefix and few blocks: each reads the prefix for itself, which saves the
    // second launch and the shares (8-bit, 140 keys of their own, alone against shared:
    // 16 sequences of 3 rows on 4 heads, prefix 256: 7.9 us against 13.0, 600: 10.6
    // against 13.4, 1500: 14.5 against 13.5; 64 sequences on 8 heads, 600: 13.5 against
    // 14.3, 1000: 15.5 against 14.1; 256 sequences, 2048 blocks, 256: 25.1 against 22.5).
    if (prefix_length > 0 && (!own || own->format == prefix->format)) {
        const int few = few_rows(prefix), rows = own_rows <= few ? few : own_rows <= 16 ? 16 : 32;
        const int64_t blocks = (int64_t)sequences * kv_heads * ((own_rows + rows - 1) / rows);
        n.alone = blocks <= 2 * kCus && (int64_t)prefix_length + own_capacity / 2 <= kAloneKeys;
        if (n.alone) {
            n.qo = rows == few ? 0 : rows / 16;
            n.own_tiles = (own_rows + rows - 1) / rows;
            n.own_splits = 1;
            n.direct = true;
            return n;
        }
    }
    if (prefix_length > 0) {
        n.qp = shared_rows <= few_rows(prefix) ? 0 : shared_rows <= 16 ? 1 : 2;
        n.wp = shared_rows <= 32 ? 1 : shared_rows <= 64 ? 2 : 4;
        const int tile = n.qp == 0 ? few_rows(prefix) : 16 * n.qp * n.wp;
        n.prefix_tiles = (shared_rows + tile - 1) / tile;
        // no query sees below the first position of the first query of an empty own cache
        if (window > 0) n.prefix_first = prefix_length - queries + 1 - window > 0 ? prefix_length - queries + 1 - window : 0;
        if (n.prefix_first >= prefix_length) n.prefix_first = prefix_length - 1;
        // Blocks of the prefix: two a CU, or one where the own caches' blocks have enough
        // to do meanwhile, which fewer shares to join then repay (256 rows over 32768
        // positions and 550 of their own, 8-bit: 79 us with two, 75 with one; without own
        // caches 61 and 72; 480 rows over 4096: 23 and 20); each of two rounds at least,
        // four beside the blocks of own caches.
        const int keys = prefix_length - n.prefix_first, base = kv_heads * n.prefix_tiles;
        const int round = kRoundKeys * (4 / n.wp), rounds = (keys + round - 1) / round;
        const int64_t mine = (int64_t)base * rounds, theirs = (int64_t)sequences * kv_heads * own_capacity / kOwnKeys;
        const int blocks = mine > 32 * kCus && theirs < mine / 4 ? 2 * kCus : kCus;
        const int splits = (blocks + base - 1) / base, fewest = own_capacity > 0 ? 4 : 2;
        const int most = (rounds + fewest - 1) / fewest;
        n.prefix_splits = splits > most ? most : splits;
    }
    if (own_capacity > 0) {
        n.qo = own_rows <= few_rows(own) ? 0 : own_rows <= 16 ? 1 : 2;
        const int tile = n.qo == 0 ? few_rows(own) : 16 * n.qo;
        n.own_tiles = (own_rows + tile - 1) / tile;
        const int keys = (own_capacity + 63) / 64, most = (keys + 3) / 4;
        const int64_t base = (int64_t)sequences * kv_heads * n.own_tiles;
        const int64_t splits = (2 * kCus + base - 1) / base;
        n.own_splits = (int)(splits > most ? most : splits);
    }
    const int slots = n.prefix_splits + n.own_splits;
    n.direct = slots == 1 && n.prefix_splits == 0;
    n.stats_at = aligned_bytes((size_t)slots * n.rows * kCacheWidth * 4);
    n.bytes = n.direct ? 0 : n.stats_at + aligned_bytes((size_t)slots * n.rows * 8);
    return n;
}

template <bool I8, int QP, int WP>
void launch_with(const Plan& n, const SharedParams& p, hipStream_t s) {
    const dim3 grid(p.prefix_tasks + p.own_tasks), block(256);
    if (n.qo == 0) {
        rn_launch(shared_attend_kernel<I8, QP, WP, 0>, grid, block, 0, s, p);
        return;
    }
    if constexpr (QP > 0) {  // an own cache has no more rows than the prefix
        if (n.qo == 1) {
            rn_launch(shared_attend_kernel<I8, QP, WP, 1>, grid, block, 0, s, p);
            return;
        }
    }
    if constexpr (QP > 1) rn_launch(shared_attend_kernel<I8, QP, WP, 2>, grid, block, 0, s, p);
}

template <bool I8>
void launch_alone(const Plan& n, const SharedParams& p, hipStream_t s) {
    const dim3 grid(p.sequences * p.kv_heads * n.own_tiles), block(256);
    if (n.qo == 0)
        rn_launch(alone_attend_kernel<I8, 0>, grid, block, 0, s, p);
    else if (n.qo == 1)
        rn_launch(alone_attend_kernel<I8, 1>, grid, block, 0, s, p);
    else
        rn_launch(alone_attend_kernel<I8, 2>, grid, block, 0, s, p);
}

template <bool I8>
void launch(const Plan& n, const SharedParams& p, hipStream_t s) {
    if (n.qp == 0 && n.qo == 0)
        launch_with<I8, 0, 1>(n, p, s);
    else if (n.qp <= 1 && n.qo <= 1)
        launch_with<I8, 1, 1>(n, p, s);
    else if (n.wp == 1)
        launch_with<I8, 2, 1>(n, p, s);
    else if (n.wp == 2)
        launch_with<I8, 2, 2>(n, p, s);
    else
        launch_with<I8, 2, 4>(n, p, s);
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
        *bytes = plan_of(sequences, queries, heads, prefix, prefix_length, own, 0).bytes;
    return RN_OK;
}

int rn_attend_shared(const float* q, int64_t q_stride, float* out, int64_t out_stride, int sequences, int queries,
                     int heads, const rn_cache* prefix, int prefix_length, const rn_cache* own,
                     const int32_t* lengths, const int32_t* counts, float scale, int window, void* workspace,
                     size_t workspace_bytes, int32_t* error, void* stream) {
    int kv_heads, capacity;
    SV_CHECK(check_shape(sequences, queries, heads, prefix, prefix_length, own, kv_heads, capacity));
    SV_REQUIRE(own || !lengths, "lengths without an own cache");
    const float scale2 = scale * 1.44269504088896340736f;
    SV_REQUIRE(scale > 0.0f && scale2 < INFINITY, "scale must be positive and below 2.3e38");
    SV_REQUIRE(window >= 0, "window must not be negative (got %d)", window);
    if (window > (1 << 26)) window = 0;  // wider than any sequence
    if (sequences == 0 || queries == 0) return RN_OK;
    SV_REQUIRE(q && out, "null argument");
    SV_REQUIRE(q_stride >= (int64_t)heads * kCacheWidth && out_stride >= (int64_t)heads * kCacheWidth &&
                   q_stride % 4 == 0 && out_stride % 4 == 0 && q_stride <= ((int64_t)1 << 40) &&
                   out_stride <= ((int64_t)1 << 40),
               "q_stride and out_stride must be multiples of 4 that hold a row of %d floats", heads * kCacheWidth);
    const Plan n = plan_of(sequences, queries, heads, prefix, prefix_length, own, window);
    const size_t needed = plan_of(sequences, queries, heads, prefix, prefix_length, own, 0).bytes;
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
    SV_CHECK(on.optional(workspace, 256, "workspace"));

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
    p.scale2 = scale2;
    const int64_t shared = (int64_t)kv_heads * n.prefix_tiles * n.prefix_splits;
    const int64_t single = (int64_t)sequences * kv_heads * n.own_tiles * n.own_splits;
    hipStream_t s = (hipStream_t)stream;
    const bool mixed = prefix_length > 0 && own && prefix->format != own->format;
    // one launch for both kinds of blocks, or one each where the caches' formats differ
    if (n.alone) {
        prefix->format == RN_CACHE_I8 ? launch_alone<true>(n, p, s) : launch_alone<false>(n, p, s);
        SV_HIP(hipGetLastError());
    } else if (prefix_length > 0) {
        p.prefix_tasks = (int)shared;
        p.own_tasks = mixed ? 0 : (int)single;
        prefix->format == RN_CACHE_I8 ? launch<true>(n, p, s) : launch<false>(n, p, s);
        SV_HIP(hipGetLastError());
    }
    if (own && !n.alone && (mixed || prefix_length == 0)) {
        p.prefix_tasks = 0;
        p.own_tasks = (int)single;
        own->format == RN_CACHE_I8 ? launch<true>(n, p, s) : launch<false>(n, p, s);
        SV_HIP(hipGetLastError());
    }
    if (!n.direct) {
        rn_launch(shared_join_kernel, dim3((n.rows + 3) / 4), dim3(256), 0, s, p);
        SV_HIP(hipGetLastError());
    }
    return RN_OK;
}
