// rn_verify.hip — verification of drafted tokens against the target's probabilities
// from given uniforms (rn_verify_drafts).
//
// With p_i = softmax(target_i / T) and q_i = softmax(draft_i / T) (all of it on the
// drafted token where there are no draft logits), drafted token x_i is accepted while
// u_i q_i(x_i) < p_i(x_i); at the first refusal i the sequence goes on with a token of
// max(0, p_i - q_i) (of p_i where that is zero everywhere), after the last accepted
// one with a token of p_count. A token is drawn by inversion: the first index whose
// running sum passes u times the total.
//
// The border of a draw lies between sums of thousands of weights: in 32 bits about one
// draw in a hundred would depend on the order of additions. The logits are read in 32
// bits, and exponentials, sums and the comparison are 64-bit, so that the answer is the
// formula's. A weight and its sum are 16 instructions, at the full rate of this chip's
// vector units, which keeps the pass over the logits bound by memory: 285 MB, 64
// sequences of 8 drafts over 65536, in 55 us (5.2 TB/s; a copy reaches 4.9).
//
// First every row's maximum and sum by chunks (the only pass over all rows), then the
// accepted run and the draw: one block a sequence for vocabularies up to 8192, else
// the run and the chunk sums of the one row that is drawn from, and the draw's chunk
// and index in a third launch.
#include "rn_device.hpp"
#include "rn_serving.hpp"

namespace rn {
namespace {

constexpr int kThreads = 256;

struct VerifyParams {
    const float* target;  // [sequences][drafts + 1] rows, target_stride floats apart
    const float* draft;   // [sequences][drafts] rows, or null
    int64_t target_stride, draft_stride;
    const int32_t* tokens;  // [sequences][drafts]
    const int32_t* counts;
    const float* temperatures;
    const float* uniforms;  // [sequences][drafts + 1]: of each drafted token, then of the draw
    int32_t* accepted;
    int32_t* emitted;       // [sequences][drafts + 1]
    float* probabilities;
    int32_t* error;
    struct RowPart* parts;   // [sequences][rows a sequence][row_parts]
    double2* sums;           // [sequences][chunks]: of the drawn row's rest, and of p
    struct Verdict* verdicts;  // [sequences]
    int sequences, drafts, vocab, rows, row_parts, chunks, span;
};

// One chunk of one row: the sum of exp((x - peak) / T), the peak; at temperature 0 the
// greedy key instead of the sum. bad: a NaN or +infinity.
struct RowPart {
    union {
        double sum;
        uint64_t key;
    };
    float peak;
    int32_t bad;
};

// What the draw needs to know of its sequence.
struct Verdict {
    double p_scale, ratio;  // 1 / sum of the target's row; sum of it over that of the draft's
    float p_peak, q_peak;
    int32_t at;       // accepted tokens; the row of the draw
    int32_t refused;  // the rest of row `at` is drawn from, not all of it
    int32_t choice;   // >= 0: the token (greedy); -1: to be drawn; -2: none, its numbers are bad
    int32_t spare;
};

constexpr double kLog2e = 1.4426950408889634;

// exp((x - peak) / T) with warm = log2(e) / T and least = least_of(temperature). What is less
// than 2^-1000, a masked logit among it, comes out as 2^-1000, which no sum of a row
// notices (its peak's is 1); a weight counts from kLeast on.
// 2^y, y = (x - peak) warm, relative error below 1.1e-12: y = n + r, |r| <= 1/2, 2^r by
// its interpolation of degree 8 at the Chebyshev nodes of that interval (exact at 0);
// n is the low bits of y + 1.5 2^52. 15 instructions with the sum's (v_ldexp_f64
// instead of an addition to the exponent, which took five, and y never by itself: 20
// before that, and the pass over 64 x 17 rows of 65536 63 us, 59 then).
__device__ __forceinline__ double least_of(float temperature) { return -1000.0 / kLog2e * (double)temperature; }
__device__ __forceinline__ double weight(float x, double peak, double warm, double least) {
    const double d = __builtin_fmax((double)x - peak, least);
    const double t = __builtin_fma(d, warm, 0x1.8p+52), r = __builtin_fma(d, warm, -(t - 0x1.8p+52));
    double p = 0x1.63d1363a681b4p-20;
    p = __builtin_fma(p, r, 0x1.00dc4a5344ef5p-16);
    p = __builtin_fma(p, r, 0x1.4308ac85a69f8p-13);
    p = __builtin_fma(p, r, 0x1.5d8745a728209p-10);
    p = __builtin_fma(p, r, 0x1.3b2ab7181b77dp-7);
    p = __builtin_fma(p, r, 0x1.c6b08dd6fd236p-5);
    p = __builtin_fma(p, r, 0x1.ebfbdff823cedp-3);
    p = __builtin_fma(p, r, 0x1.62e42fef84cf0p-1);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_ldexp(p, (int)(uint32_t)(uint64_t)__double_as_longlong(t));
}
constexpr double kLeast = 0x1p-990;  // of one index; 2^24 masked ones sum up to less than kMost
constexpr double kMost = 0x1p-970;
__device__ __forceinline__ double likely(float x, double peak, double warm, double least) {
    const double w = weight(x, peak, warm, least);
    return w < kLeast ? 0.0 : w;
}

__device__ __forceinline__ double of_halves(uint32_t lo, uint32_t hi) {
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return of_halves((uint32_t)dpp_move<CTRL>((int)(uint32_t)u), (uint32_t)dpp_move<CTRL>((int)(uint32_t)(u >> 32)));
}
// The sum over each run of 8 lanes, in all of them.
__device__ __forceinline__ double row8_sum(double v) {
    v += dpp_f64<0xb1>(v);
    v += dpp_f64<0x4e>(v);
    return v + dpp_f64<0x141>(v);
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    return __longlong_as_double((long long)lane_u64((uint64_t)__double_as_longlong(v), lane));
}
__device__ __forceinline__ double wave_sum(double v) {
    v = row8_sum(v);
    v += dpp_f64<0x140>(v);
    return (lane_f64(v, 0) + lane_f64(v, 16)) + (lane_f64(v, 32) + lane_f64(v, 48));
}
__device__ __forceinline__ float row8_max(float v) {
    v = fmaxf(v, __int_as_float(dpp_move<0xb1>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(dpp_move<0x4e>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(dpp_move<0x141>(__float_as_int(v))));
}
// The sum of this lane's and all lower lanes' values: in each row of 16 lanes by row
// shifts (a lane without a source adds 0), then the rows below.
template <int SHIFT>
__device__ __forceinline__ double row_shift_f64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return of_halves((uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, 0x110 + SHIFT, 0xf, 0xf, true),
                     (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), 0x110 + SHIFT, 0xf, 0xf, true));
}
__device__ __forceinline__ double wave_scan(double v) {
    v += row_shift_f64<1>(v);
    v += row_shift_f64<2>(v);
    v += row_shift_f64<4>(v);
    v += row_shift_f64<8>(v);
    const double a = lane_f64(v, 15), b = a + lane_f64(v, 31), c = b + lane_f64(v, 47);
    const int row = threadIdx.x % 64 / 16;
    return v + (row == 0 ? 0.0 : row == 1 ? a : row == 2 ? b : c);
}

// Four consecutive logits of a row at i (-infinity past its end); rows need no more
// than the alignment of a float.
__device__ __forceinline__ void load_logits(const float* row, int i, int vocab, float* x) {
    typedef float v4u __attribute__((ext_vector_type(4), aligned(4)));
    if (i + 4 <= vocab) {
        const v4u t = *reinterpret_cast<const v4u*>(row + i);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = t[c];
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = i + c < vocab ? row[i + c] : -__builtin_inff();
    }
}

// Row r of sequence b: 0..drafts the target's, drafts + 1.. the draft's.
__device__ __forceinline__ const float* row_of(const VerifyParams& p, int b, int r) {
    return r <= p.drafts ? p.target + (int64_t)(b * (p.drafts + 1) + r) * p.target_stride
                         : p.draft + (int64_t)(b * p.drafts + r - p.drafts - 1) * p.draft_stride;
}

// A sequence's drafted tokens, -1 where count or temperature is out of range.
__device__ __forceinline__ int count_of(const VerifyParams& p, int b, float& temperature) {
    const int count = p.counts ? p.counts[b] : p.drafts;
    temperature = p.temperatures ? p.temperatures[b] : 1.0f;
    return count < 0 || count > p.drafts || !(temperature >= 0.0f && temperature < __builtin_inff()) ? -1 : count;
}

template <int E>
__global__ __launch_bounds__(kThreads) void verify_rows_kernel(const VerifyParams p) {
    const int chunk = blockIdx.x, r = blockIdx.y, b = blockIdx.z, t = threadIdx.x;
    float temperature;
    const int count = count_of(p, b, temperature);
    if (r > p.drafts ? r - p.drafts - 1 >= count : r > count) return;  // a row that no token needs
    const float* row = row_of(p, b, r);
    float x[E][4];
#pragma unroll
    for (int e = 0; e < E; ++e) load_logits(row, (chunk * E + e) * kThreads * 4 + t * 4, p.vocab, x[e]);
    float peak = -__builtin_inff();
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            peak = __builtin_elementwise_maximum(peak, x[e][c]);
        }
    __shared__ float peaks[4];
    __shared__ double sums[4];
    __shared__ uint64_t keys[4];
    __shared__ int bads[4];
    const int wave = t / 64;
    const bool bad = !(peak < __builtin_inff());  // a NaN wins
    peak = wave_max(peak);
    if (t % 64 == 0) peaks[wave] = peak;
    __syncthreads();
    peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
    double sum = 0.0;
    uint64_t key = 0;
    if (temperature > 0.0f) {
        // a chunk of masked logits has no sum; elsewhere their 2^-1000 do not matter
        if (peak > -__builtin_inff()) {
            const double warm = kLog2e / (double)temperature, least = least_of(temperature);
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) sum += weight(x[e][c], (double)peak, warm, least);
            sum = wave_sum(sum);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint64_t k = argmax_key(x[e][c], (uint32_t)((chunk * E + e) * kThreads * 4 + t * 4 + c));
                key = k > key ? k : key;
            }
        key = wave_max_u64(key);
    }
    const bool any = __any(bad);
    if (t % 64 == 0) {
        sums[wave] = sum;
        keys[wave] = key;
        bads[wave] = any;
    }
    __syncthreads();
    if (t == 0) {
        RowPart out;
        if (temperature > 0.0f) {
            out.sum = ((sums[0] + sums[1]) + sums[2]) + sums[3];
        } else {
            for (int w = 1; w < 4; ++w) key = keys[w] > key ? keys[w] : key;
            out.key = key;
        }
        out.peak = peak;
        out.bad = bads[0] | bads[1] | bads[2] | bads[3];
        p.parts[((int64_t)b * p.rows + r) * p.row_parts + chunk] = out;
    }
}

constexpr int kMaxDrafts = 63;  // a lane each, and one for the draw

// The weights of the draw at four logits, times the sum of the target's row: what is
// left of p, and p.
struct Draw {
    double warm, least, p_peak, q_peak, ratio;
    const float* p_row;
    const float* q_row;  // null: nothing is taken off but `token`
    int token;           // taken off p where there are no draft logits; -1: none
    int vocab;

    __device__ __forceinline__ void load(int i, float* x, float* y) const {
        load_logits(p_row, i, vocab, x);
        if (q_row) load_logits(q_row, i, vocab, y);
    }
    __device__ __forceinline__ void at(int i, double* rest, double* all) const {
        float x[4], y[4];
        load(i, x, y);
        of(i, x, y, rest, all);
    }
    __device__ __forceinline__ void of(int i, const float* x, const float* y, double* rest, double* all) const {
#pragma unroll
        for (int c = 0; c < 4; ++c) rest[c] = all[c] = weight(x[c], p_peak, warm, least);
        if (q_row) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                rest[c] = __builtin_fmax(__builtin_fma(-weight(y[c], q_peak, warm, least), ratio, all[c]), 0.0);
        } else if (token >= 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (i + c == token) rest[c] = 0.0;
        }
    }
};

__device__ __forceinline__ Draw draw_of(const VerifyParams& p, int b, const Verdict& v, float temperature) {
    Draw d;
    d.warm = kLog2e / (double)temperature;
    d.least = least_of(temperature);
    d.p_peak = (double)v.p_peak;
    d.q_peak = (double)v.q_peak;
    d.ratio = v.ratio;
    d.p_row = row_of(p, b, v.at);
    d.q_row = v.refused && p.draft ? row_of(p, b, p.drafts + 1 + v.at) : nullptr;
    d.token = v.refused && !p.draft ? p.tokens[b * p.drafts + v.at] : -1;
    d.vocab = p.vocab;
    return d;
}

struct Rows {
    double totals[2 * kMaxDrafts + 1], inverse[2 * kMaxDrafts + 1];  // sum of the row's weights, 1 / it
    float peaks[2 * kMaxDrafts + 1];
    int firsts[2 * kMaxDrafts + 1];  // greedy: the first largest index; -1: the row is bad
    Verdict verdict;
};

// The accepted run of a sequence, by a whole block; with `tell` it is written down.
template <int THREADS>
__device__ __forceinline__ Verdict judge(const VerifyParams& p, int b, float& temperature, Rows& rows, bool tell) {
    const int t = threadIdx.x, lane = t % 64, wave = t / 64;
    // what lane i needs of drafted token i, asked for before anything is waited for
    int token = -1;
    float u = 0.0f, x = 0.0f, y = 0.0f;
    const bool mine = wave == 0 && lane < p.drafts;
    if (mine) {
        token = p.tokens[b * p.drafts + lane];
        u = p.uniforms[b * (p.drafts + 1) + lane];
    }
    const int count = count_of(p, b, temperature);
    const bool greedy = !(temperature > 0.0f);
    if (mine && token >= 0 && token < p.vocab) {
        x = row_of(p, b, lane)[token];
        if (p.draft) y = row_of(p, b, p.drafts + 1 + lane)[token];
    }
    const double warm = greedy ? 1.0 : kLog2e / (double)temperature, least = least_of(temperature);
    // ---- every row's total, eight lanes a row
    for (int r = t / 8; r < p.rows; r += THREADS / 8) {
        if (r > p.drafts ? r - p.drafts - 1 >= count : r > count) continue;
        const RowPart* parts = p.parts + ((int64_t)b * p.rows + r) * p.row_parts;
        float peak = -__builtin_inff();
        double total = 0.0;
        int bad = 0;
        uint64_t key = 0;
#pragma unroll 2
        for (int c = lane % 8; c < p.row_parts; c += 8) {
            const RowPart part = parts[c];
            bad |= part.bad;
            if (greedy) {
                key = part.key > key ? part.key : key;
                peak = fmaxf(peak, part.peak);
            } else if (part.peak > peak) {
                total = total * likely(peak, part.peak, warm, least) + part.sum;
                peak = part.peak;
            } else if (part.peak > -__builtin_inff()) {
                total += part.sum * likely(part.peak, peak, warm, least);
            }
        }
        const float most = row8_max(peak);
        bad |= dpp_move<0xb1>(bad);
        bad |= dpp_move<0x4e>(bad);
        bad |= dpp_move<0x141>(bad);
        if (greedy) {
            key = max_with_dpp_u64<0xb1>(key);
            key = max_with_dpp_u64<0x4e>(key);
            key = max_with_dpp_u64<0x141>(key);
        } else {
            total = row8_sum(peak > -__builtin_inff() ? total * likely(peak, most, warm, least) : 0.0);
        }
        if (lane % 8 == 0) {
            rows.totals[r] = total;
            rows.inverse[r] = 1.0 / total;
            rows.peaks[r] = most;
            rows.firsts[r] = bad || !(most > -__builtin_inff()) ? -1 : greedy ? (int)argmax_index(key) : 0;
        }
    }
    __syncthreads();
    // ---- the accepted run: lane i judges drafted token i, lane `count` the draw's row
    if (wave == 0) {
        int state = 0;  // 0 accepted, 1 the run ends here, 2 it cannot be judged
        double chance = 0.0;  // of the drafted token, under the target
        if (count < 0) {
            state = 2;
        } else if (lane <= count) {
            if (rows.firsts[lane] < 0) {
                state = 2;
            } else if (lane == count) {
                state = 1;
            } else {
                const int dr = p.drafts + 1 + lane;
                if (token < 0 || token >= p.vocab || (p.draft && rows.firsts[dr] < 0)) {
                    state = 2;
                } else if (greedy) {
                    chance = token == rows.firsts[lane] ? 1.0 : 0.0;
                    state = token == rows.firsts[lane] ? 0 : 1;
                } else {
                    chance = likely(x, rows.peaks[lane], warm, least) * rows.inverse[lane];
                    double q = 1.0;
                    if (p.draft) q = likely(y, rows.peaks[dr], warm, least) * rows.inverse[dr];
                    state = (double)u * q < chance ? 0 : 1;
                }
            }
        } else {
            state = 1;
        }
        const uint64_t ends = __ballot(state != 0);
        const int at = __builtin_ctzll(ends);  // count <= 63: some lane ends the run
        const int end = __shfl(state, at);
        if (tell) {
            if (lane < at) {
                p.emitted[b * (p.drafts + 1) + lane] = token;
                if (p.probabilities) p.probabilities[b * (p.drafts + 1) + lane] = (float)chance;
            }
            if (lane == 0) {
                p.accepted[b] = at;
                if (end == 2) {
                    p.emitted[b * (p.drafts + 1) + at] = -1;
                    if (p.probabilities) p.probabilities[b * (p.drafts + 1) + at] = 0.0f;
                    if (p.error) *p.error = RN_ERR_ARGUMENT;
                } else if (greedy) {
                    p.emitted[b * (p.drafts + 1) + at] = rows.firsts[at];
                    if (p.probabilities) p.probabilities[b * (p.drafts + 1) + at] = 1.0f;
                }
            }
        }
        if (lane == 0) {
            Verdict v{};
            v.at = at;
            v.refused = at < count;
            v.choice = end == 2 ? -2 : greedy ? rows.firsts[at] : -1;
            if (v.choice == -1) {
                v.p_scale = rows.inverse[at];
                v.p_peak = rows.peaks[at];
                if (v.refused && p.draft) {
                    v.ratio = rows.totals[at] / rows.totals[p.drafts + 1 + at];  // 1 for equal rows
                    v.q_peak = rows.peaks[p.drafts + 1 + at];
                }
            }
            rows.verdict = v;
        }
    }
    __syncthreads();
    return rows.verdict;
}

// The draw among this block's 4 E THREADS consecutive weights w from `first` on (each
// thread its run of 4 E, their sum `mine`, `upto` that of the wave's lanes up to it,
// `sums` that of every wave): the first index whose running sum, `base` before them,
// is above `border`; past the end, by a rounding or by a uniform of 1, the last with a
// weight. The one thread that holds it writes it down, with its weight under the target.
template <int THREADS, int E>
__device__ __forceinline__ void pick(const VerifyParams& p, int b, const Verdict& v, const double (&w)[E][4],
                                     const double (&all)[E][4], double mine, double upto, const double* sums,
                                     double base, double border, int first) {
    const int t = threadIdx.x, lane = t % 64, wave = t / 64;
    // every wave finds the wave, that one the lane, that one the index
    int chosen = -1;
    double below = base, mark = base;
    for (int k = 0; k < THREADS / 64; ++k) {
        const double s = sums[k];
        if (s > kMost) {
            chosen = k;
            mark = below;
            if (below + s > border) break;
        }
        below += s;
    }
    if (wave != chosen) return;
    const uint64_t over = __ballot(mine > kMost && mark + upto > border), some = __ballot(mine > kMost);
    if (some == 0 || lane != (over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some))) return;
    double sum = mark + (upto - mine), chance = 0.0;
    int token = -1;
    bool done = false;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (w[e][c] > kLeast && !done) {
                sum += w[e][c];
                token = first + 4 * e + c;
                chance = all[e][c];
                done = sum > border;
            }
    const int at = b * (p.drafts + 1) + v.at;
    p.emitted[at] = token;
    if (p.probabilities) p.probabilities[at] = (float)(chance * v.p_scale);
}

constexpr int kWide = 1024;  // threads of a block that holds a whole row

// The accepted run and the draw of a sequence whose vocabulary one block holds.
template <int E>
__global__ __launch_bounds__(kWide) void verify_finish_kernel(const VerifyParams p) {
    const int b = blockIdx.x, t = threadIdx.x, lane = t % 64, wave = t / 64;
    __shared__ Rows rows;
    __shared__ double rests[kWide / 64], wholes[kWide / 64];
    float temperature;
    const float u = p.uniforms[b * (p.drafts + 1) + p.drafts];
    const Verdict v = judge<kWide>(p, b, temperature, rows, true);
    if (v.choice != -1) return;
    const Draw d = draw_of(p, b, v, temperature);
    double w[E][4], a[E][4], mine = 0.0;
    const int first = t * E * 4;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        d.at(first + 4 * e, w[e], a[e]);
#pragma unroll
        for (int c = 0; c < 4; ++c) mine += w[e][c];
    }
    double upto = wave_scan(mine);
    if (lane == 63) rests[wave] = upto;
    __syncthreads();
    double total = 0.0;
    double* sums = rests;
    for (int k = 0; k < kWide / 64; ++k) total += rests[k];
    if (!(total > kMost)) {  // nothing is left of p: all of it
        mine = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                w[e][c] = a[e][c];
                mine += a[e][c];
            }
        upto = wave_scan(mine);
        if (lane == 63) wholes[wave] = upto;
        __syncthreads();
        total = 0.0;
        for (int k = 0; k < kWide / 64; ++k) total += wholes[k];
        sums = wholes;
    }
    pick<kWide, E>(p, b, v, w, a, mine, upto, sums, 0.0, (double)u * total, first);
}

constexpr int kSpan = 8;  // most chunks a block

// The accepted run of a sequence (every block of it finds the same), and the sums of
// this block's chunks, four logits a thread, of the row that is drawn from. Few blocks
// of several chunks, the next one's logits asked for in time: judged in a launch of its
// own, with a block a chunk after it, the two took 17.7 us for 64 sequences of 65536.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void verify_run_kernel(const VerifyParams p) {
    const int b = blockIdx.y, t = threadIdx.x, lane = t % 64, wave = t / 64;
    const int c0 = blockIdx.x * p.span, c1 = min(c0 + p.span, p.chunks);
    __shared__ Rows rows;
    __shared__ double2 sums[kSpan][THREADS / 64];
    float temperature;
    const Verdict v = judge<THREADS>(p, b, temperature, rows, c0 == 0);
    if (c0 == 0 && t == 0) p.verdicts[b] = v;
    if (v.choice != -1) return;
    const Draw d = draw_of(p, b, v, temperature);
    float x[4], y[4];
    d.load((c0 * THREADS + t) * 4, x, y);
#pragma unroll 1
    for (int c = c0; c < c1; ++c) {
        double r4[4], a4[4];
        const float x0[4] = {x[0], x[1], x[2], x[3]}, y0[4] = {y[0], y[1], y[2], y[3]};
        if (c + 1 < c1) d.load(((c + 1) * THREADS + t) * 4, x, y);
        d.of((c * THREADS + t) * 4, x0, y0, r4, a4);
        const double rest = wave_sum((r4[0] + r4[1]) + (r4[2] + r4[3])), all = wave_sum((a4[0] + a4[1]) + (a4[2] + a4[3]));
        if (lane == 0) sums[c - c0][wave] = make_double2(rest, all);
    }
    __syncthreads();
    if (t < c1 - c0) {
        double2 s = sums[t][0];
        for (int k = 1; k < THREADS / 64; ++k) {
            s.x += sums[t][k].x;
            s.y += sums[t][k].y;
        }
        p.sums[(int64_t)b * p.chunks + c0 + t] = s;
    }
}

// The draw: the chunk whose running sum passes u times the total, and in it the index.
// Every wave finds the chunk by itself, a lane a chunk. (A launch of its own, 7 us; done
// by the last block of a sequence in the launch before, that took 47 us instead of 14:
// every block's arrival writes back and empties its L2.)
template <int THREADS>
__global__ __launch_bounds__(THREADS) void verify_draw_kernel(const VerifyParams p) {
    const int b = blockIdx.x, t = threadIdx.x, lane = t % 64, wave = t / 64;
    const float u = p.uniforms[b * (p.drafts + 1) + p.drafts];
    const float temperature = p.temperatures ? p.temperatures[b] : 1.0f;
    const double2* sums = p.sums + (int64_t)b * p.chunks;
    const Verdict v = p.verdicts[b];
    if (v.choice != -1) return;
    __shared__ double waves[THREADS / 64];
    double rest = 0.0, all = 0.0;
    for (int c = lane; c < p.chunks; c += 64) {
        const double2 s = sums[c];
        rest += s.x;
        all += s.y;
    }
    rest = wave_sum(rest);
    const bool whole = !(rest > kMost);  // nothing is left of p: all of it
    const double border = (double)u * (whole ? wave_sum(all) : rest);
    double base = 0.0, running = 0.0;
    int chunk = 0;
    for (int c0 = 0; c0 < p.chunks; c0 += 64) {
        double s = 0.0;
        if (c0 + lane < p.chunks) s = whole ? sums[c0 + lane].y : sums[c0 + lane].x;
        const double upto = running + wave_scan(s);
        const uint64_t over = __ballot(s > kMost && upto > border), some = __ballot(s > kMost);
        // the first chunk that passes the border, or the last with a weight so far
        const int at = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
        if (at >= 0) {
            chunk = c0 + at;
            base = lane_f64(upto, at) - lane_f64(s, at);
        }
        if (over) break;
        running = lane_f64(upto, 63);
    }
    const Draw d = draw_of(p, b, v, temperature);
    double w[1][4], a[1][4];
    const int first = (chunk * THREADS + t) * 4;
    d.at(first, w[0], a[0]);
    if (whole) {
#pragma unroll
        for (int c = 0; c < 4; ++c) w[0][c] = a[0][c];
    }
    const double mine = (w[0][0] + w[0][1]) + (w[0][2] + w[0][3]), upto = wave_scan(mine);
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    pick<THREADS, 1>(p, b, v, w, a, mine, upto, waves, base, border, first);
}

struct VerifyPlan {
    int rows = 0, each = 1, row_parts = 0, chunks = 0;  // each: 4-logit loads a thread of the pass over all rows
    size_t sums_at = 0, verdicts_at = 0, bytes = 0;
};

VerifyPlan verify_plan(int sequences, int drafts, int vocab) {
    VerifyPlan n;
    n.rows = 2 * drafts + 1;
    // 32 logits a thread where that still gives the chip four blocks a CU, else 16, else 4:
    // a thread's joins and its 64-bit quotient are about 110 instructions (64 x 17 rows of
    // 65536: 55 us with 32, 59 with 16; 64 x 9 of 8192, too few for 32: 7.3 with 16)
    const int64_t all = (int64_t)sequences * n.rows;
    n.each = all * ((vocab + 8191) / 8192) >= 1024 ? 8 : all * ((vocab + 4095) / 4096) >= 1024 ? 4 : 1;
    n.row_parts = (vocab + 1024 * n.each - 1) / (1024 * n.each);
    n.chunks = n.each > 1 ? (vocab + 4095) / 4096 : n.row_parts;
    n.sums_at = aligned_bytes((size_t)sequences * n.rows * n.row_parts * sizeof(RowPart));
    n.verdicts_at = n.sums_at + aligned_bytes((size_t)sequences * n.chunks * sizeof(double2));
    n.bytes = n.verdicts_at + aligned_bytes((size_t)sequences * sizeof(Verdict));
    return n;
}

int check_verify(int sequences, int drafts, int vocab) {
    SV_REQUIRE(sequences >= 0 && sequences <= 65535, "sequences must be 0..65535 (got %d)", sequences);
    SV_REQUIRE(drafts >= 0 && drafts <= kMaxDrafts, "drafts must be 0..%d (got %d)", kMaxDrafts, drafts);
    SV_REQUIRE(vocab >= 1 && vocab <= 1 << 24, "vocab must be 1..2^24 (got %d)", vocab);
    return RN_OK;
}

}  // namespace
}  // namespace rn

using namespace rn;

int rn_verify_drafts_workspace(int sequences, int drafts, int vocab, size_t* bytes) {
    SV_REQUIRE(bytes, "null argument");
    SV_CHECK(check_verify(sequences, drafts, vocab));
    *bytes = sequences > 0 ? verify_plan(sequences, drafts, vocab).bytes : 0;
    return RN_OK;
}

int rn_verify_drafts(int sequences, int drafts, int vocab, const float* target, int64_t target_stride,
                     const float* draft, int64_t draft_stride, const int32_t* tokens, const int32_t* counts,
                     const float* temperatures, const float* uniforms, int32_t* accepted, int32_t* emitted,
                     float* probabilities, void* workspace, size_t workspace_bytes, int32_t* error, void* stream) {
    SV_CHECK(check_verify(sequences, drafts, vocab));
    if (sequences == 0) return RN_OK;
    SV_REQUIRE(target && uniforms && accepted && emitted && (tokens || drafts == 0), "null argument");
    SV_REQUIRE(target_stride >= vocab && target_stride <= ((int64_t)1 << 40) &&
                   (!draft || (draft_stride >= vocab && draft_stride <= ((int64_t)1 << 40))),
               "row strides must hold the %d logits of a row", vocab);
    if (drafts == 0) draft = nullptr;
    const VerifyPlan n = verify_plan(sequences, drafts, vocab);
    SV_REQUIRE(workspace && workspace_bytes >= n.bytes, "the workspace holds %zu bytes of %zu",
               workspace ? workspace_bytes : (size_t)0, n.bytes);
    OnDevice on;
    SV_CHECK(on.enter((hipStream_t)stream));
    SV_CHECK(on.pointer(target, 4, "target"));
    SV_CHECK(on.optional(draft, 4, "draft"));
    if (drafts > 0) SV_CHECK(on.pointer(tokens, 4, "tokens"));
    SV_CHECK(on.optional(counts, 4, "counts"));
    SV_CHECK(on.optional(temperatures, 4, "temperatures"));
    SV_CHECK(on.pointer(uniforms, 4, "uniforms"));
    SV_CHECK(on.pointer(accepted, 4, "accepted"));
    SV_CHECK(on.pointer(emitted, 4, "emitted"));
    SV_CHECK(on.optional(probabilities, 4, "probabilities"));
    SV_CHECK(on.optional(error, 4, "error"));
    SV_CHECK(on.pointer(workspace, 256, "workspace"));
    VerifyParams p{};
    p.target = target;
    p.draft = draft;
    p.target_stride = target_stride;
    p.draft_stride = draft_stride;
    p.tokens = tokens;
    p.counts = counts;
    p.temperatures = temperatures;
    p.uniforms = uniforms;
    p.accepted = accepted;
    p.emitted = emitted;
    p.probabilities = probabilities;
    p.error = error;
    p.parts = (RowPart*)workspace;
    p.sums = (double2*)((char*)workspace + n.sums_at);
    p.verdicts = (Verdict*)((char*)workspace + n.verdicts_at);
    p.sequences = sequences;
    p.drafts = drafts;
    p.vocab = vocab;
    p.rows = draft ? n.rows : drafts + 1;
    p.row_parts = n.row_parts;
    p.chunks = n.chunks;
    // as many chunks a block as leave a block a CU: each block judges the run again
    const int64_t span = (int64_t)sequences * n.chunks / 256;
    p.span = span < 1 ? 1 : span > kSpan ? kSpan : (int)span;
    hipStream_t s = (hipStream_t)stream;
    const dim3 rows(n.row_parts, p.rows, sequences), run((n.chunks + p.span - 1) / p.span, sequences), draw(sequences), block(kThreads);
    rn_launch(n.each == 8   ? verify_rows_kernel<8>
              : n.each == 4 ? verify_rows_kernel<4>
                            : verify_rows_kernel<1>,
              rows, block, 0, s, p);
    if (vocab <= kWide * 8) {
        rn_launch(vocab <= kWide * 4 ? verify_finish_kernel<1> : verify_finish_kernel<2>, draw, dim3(kWide), 0, s, p);
    } else if (n.each > 1) {
        rn_launch(verify_run_kernel<4 * kThreads>, run, dim3(4 * kThreads), 0, s, p);
        rn_launch(verify_draw_kernel<4 * kThreads>, draw, dim3(4 * kThreads), 0, s, p);
    } else {
        rn_launch(verify_run_kernel<kThreads>, run, block, 0, s, p);
        rn_launch(verify_draw_kernel<kThreads>, draw, block, 0, s, p);
    }
    SV_HIP(hipGetLastError());
    return RN_OK;
}
