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
// bits, and exponentials, sums and the comparison are 64-bit (a 64-bit exponential of
// 18 operations at the full rate of this chip's vector units), so that the answer is
// the formula's.
//
// Three launches: every row's maximum and sum by chunks (the only pass over all rows);
// the accepted run and the chunk sums of the one row that is drawn from; the chunk and
// index of the draw.
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
    struct RowPart* parts;   // [sequences][rows a sequence][chunks]
    double2* sums;           // [sequences][chunks]: of the drawn row's rest, and of p
    struct Verdict* verdicts;  // [sequences]
    int sequences, drafts, vocab, rows, chunks;
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
    double p_scale, q_scale;  // 1 / total of the target's and the draft's row
    float p_peak, q_peak;
    int32_t at;       // accepted tokens; the row of the draw
    int32_t refused;  // the rest of row `at` is drawn from, not all of it
    int32_t choice;   // >= 0: the token (greedy); -1: to be drawn; -2: none, its numbers are bad
    int32_t spare;
};

// exp(x) for x <= 0, relative error below 1e-13: x = n ln2 + r, |r| <= ln2 / 2, the
// series of exp(r) to r^10 (the next term is at most 2.2e-13), times 2^n.
__device__ __forceinline__ double exp64(double x) {
    const double n = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(n, -0x1.62e42fefa39efp-1, x);
    r = __builtin_fma(n, -0x1.abc9e3b39803fp-56, r);
    double y = 1.0 / 3628800.0;
    y = __builtin_fma(y, r, 1.0 / 362880.0);
    y = __builtin_fma(y, r, 1.0 / 40320.0);
    y = __builtin_fma(y, r, 1.0 / 5040.0);
    y = __builtin_fma(y, r, 1.0 / 720.0);
    y = __builtin_fma(y, r, 1.0 / 120.0);
    y = __builtin_fma(y, r, 1.0 / 24.0);
    y = __builtin_fma(y, r, 1.0 / 6.0);
    y = __builtin_fma(y, r, 0.5);
    y = __builtin_fma(y, r, 1.0);
    y = __builtin_fma(y, r, 1.0);
    return __builtin_ldexp(y, (int)(n < -2000.0 ? -2000.0 : n));
}

// exp((x - peak) / T), 0 for a masked logit; `warm` = 1 / T.
__device__ __forceinline__ double weight(float x, float peak, double warm) {
    return x > -__builtin_inff() ? exp64(((double)x - (double)peak) * warm) : 0.0;
}

__device__ __forceinline__ double shfl_xor_f64(double v, int m) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)u, m), hi = (uint32_t)__shfl_xor((int)(uint32_t)(u >> 32), m);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double wave_sum(double v) {
    for (int m = 1; m < 64; m <<= 1) v += shfl_xor_f64(v, m);
    return v;
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
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            peak = fmaxf(peak, x[e][c]);
            bad = bad || !(x[e][c] < __builtin_inff());
        }
    __shared__ float peaks[4];
    __shared__ double sums[4];
    __shared__ uint64_t keys[4];
    __shared__ int bads[4];
    const int wave = t / 64;
    peak = wave_max(peak);
    if (t % 64 == 0) peaks[wave] = peak;
    __syncthreads();
    peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
    double sum = 0.0;
    uint64_t key = 0;
    if (temperature > 0.0f) {
        const double warm = 1.0 / (double)temperature;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c) sum += weight(x[e][c], peak, warm);
        sum = wave_sum(sum);
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
        p.parts[((int64_t)b * p.rows + r) * p.chunks + chunk] = out;
    }
}

constexpr int kMaxDrafts = 63;  // a lane each, and one for the draw

// The weights of the draw at four logits: what is left of p, and p.
struct Draw {
    double warm, p_scale, q_scale;
    float p_peak, q_peak;
    const float* p_row;
    const float* q_row;  // null: nothing is taken off but `token`
    int token;           // taken off p where there are no draft logits; -1: none
    int vocab;

    __device__ __forceinline__ void at(int i, double* rest, double* all) const {
        float x[4], y[4];
        load_logits(p_row, i, vocab, x);
        if (q_row) load_logits(q_row, i, vocab, y);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const double w = weight(x[c], p_peak, warm) * p_scale;
            double left = w;
            if (q_row) left = w - weight(y[c], q_peak, warm) * q_scale;
            if (i + c == token) left = 0.0;
            all[c] = w;
            rest[c] = left > 0.0 ? left : 0.0;
        }
    }
};

__device__ __forceinline__ Draw draw_of(const VerifyParams& p, int b, const Verdict& v, float temperature) {
    Draw d;
    d.warm = 1.0 / (double)temperature;
    d.p_scale = v.p_scale;
    d.q_scale = v.q_scale;
    d.p_peak = v.p_peak;
    d.q_peak = v.q_peak;
    d.p_row = row_of(p, b, v.at);
    d.q_row = v.refused && p.draft ? row_of(p, b, p.drafts + 1 + v.at) : nullptr;
    d.token = v.refused && !p.draft ? p.tokens[b * p.drafts + v.at] : -1;
    d.vocab = p.vocab;
    return d;
}

// The accepted run of a sequence (every block of it finds the same), and the sums of
// this block's chunk of the row that is drawn from.
template <int E>
__global__ __launch_bounds__(kThreads) void verify_run_kernel(const VerifyParams p) {
    const int chunk = blockIdx.x, b = blockIdx.y, t = threadIdx.x, lane = t % 64, wave = t / 64;
    __shared__ double totals[2 * kMaxDrafts + 1];
    __shared__ float peaks[2 * kMaxDrafts + 1];
    __shared__ int firsts[2 * kMaxDrafts + 1];  // greedy: the first largest index; -1: the row is bad
    __shared__ Verdict verdict;
    __shared__ double2 sums[4];
    float temperature;
    const int count = count_of(p, b, temperature);
    const bool greedy = !(temperature > 0.0f);
    const double warm = greedy ? 0.0 : 1.0 / (double)temperature;
    // ---- every row's total, a wave a row
    for (int r = wave; r < p.rows; r += 4) {
        if (r > p.drafts ? r - p.drafts - 1 >= count : r > count) continue;
        const RowPart* parts = p.parts + ((int64_t)b * p.rows + r) * p.chunks;
        float peak = -__builtin_inff();
        bool bad = false;
        uint64_t key = 0;
        for (int c = lane; c < p.chunks; c += 64) {
            peak = fmaxf(peak, parts[c].peak);
            bad = bad || parts[c].bad;
            if (greedy) key = parts[c].key > key ? parts[c].key : key;
        }
        peak = wave_max(peak);
        bad = __any(bad) || !(peak > -__builtin_inff());
        double total = 0.0;
        if (greedy) {
            key = wave_max_u64(key);
        } else if (!bad) {
            for (int c = lane; c < p.chunks; c += 64) total += parts[c].sum * weight(parts[c].peak, peak, warm);
            total = wave_sum(total);
        }
        if (lane == 0) {
            totals[r] = total;
            peaks[r] = peak;
            firsts[r] = bad ? -1 : greedy ? (int)argmax_index(key) : 0;
        }
    }
    __syncthreads();
    // ---- the accepted run: lane i judges drafted token i, lane `count` the draw's row
    if (wave == 0) {
        int state = 0;  // 0 accepted, 1 the run ends here, 2 it cannot be judged
        int token = -1;
        double chance = 0.0;  // of the drafted token, under the target
        if (count < 0) {
            state = 2;
        } else if (lane <= count) {
            if (firsts[lane] < 0) {
                state = 2;
            } else if (lane == count) {
                state = 1;
            } else {
                token = p.tokens[b * p.drafts + lane];
                const int dr = p.drafts + 1 + lane;
                if (token < 0 || token >= p.vocab || (p.draft && firsts[dr] < 0)) {
                    state = 2;
                } else if (greedy) {
                    chance = token == firsts[lane] ? 1.0 : 0.0;
                    state = token == firsts[lane] ? 0 : 1;
                } else {
                    const float x = row_of(p, b, lane)[token];
                    chance = weight(x, peaks[lane], warm) / totals[lane];
                    double q = 1.0;
                    if (p.draft) q = weight(row_of(p, b, dr)[token], peaks[dr], warm) / totals[dr];
                    state = (double)p.uniforms[b * (p.drafts + 1) + lane] * q < chance ? 0 : 1;
                }
            }
        } else {
            state = 1;
        }
        const uint64_t ends = __ballot(state != 0);
        const int at = __builtin_ctzll(ends);  // count <= 63: some lane ends the run
        const int end = __shfl(state, at);
        if (chunk == 0) {
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
                    p.emitted[b * (p.drafts + 1) + at] = firsts[at];
                    if (p.probabilities) p.probabilities[b * (p.drafts + 1) + at] = 1.0f;
                }
            }
        }
        if (lane == 0) {
            Verdict v{};
            v.at = at;
            v.refused = at < count;
            v.choice = end == 2 ? -2 : greedy ? firsts[at] : -1;
            if (v.choice == -1) {
                v.p_scale = 1.0 / totals[at];
                v.p_peak = peaks[at];
                if (v.refused && p.draft) {
                    v.q_scale = 1.0 / totals[p.drafts + 1 + at];
                    v.q_peak = peaks[p.drafts + 1 + at];
                }
            }
            verdict = v;
            if (chunk == 0) p.verdicts[b] = v;
        }
    }
    __syncthreads();
    const Verdict v = verdict;
    if (v.choice != -1) return;
    const Draw d = draw_of(p, b, v, temperature);
    double rest = 0.0, all = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        double r4[4], a4[4];
        d.at((chunk * E + e) * kThreads * 4 + t * 4, r4, a4);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            rest += r4[c];
            all += a4[c];
        }
    }
    rest = wave_sum(rest);
    all = wave_sum(all);
    if (lane == 0) sums[wave] = make_double2(rest, all);
    __syncthreads();
    if (t == 0)
        p.sums[(int64_t)b * p.chunks + chunk] = make_double2(((sums[0].x + sums[1].x) + sums[2].x) + sums[3].x,
                                                             ((sums[0].y + sums[1].y) + sums[2].y) + sums[3].y);
}

// The draw: the chunk whose running sum passes u times the total, and in it the index.
template <int E>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(const VerifyParams p) {
    const int b = blockIdx.x, t = threadIdx.x, lane = t % 64, wave = t / 64;
    const Verdict v = p.verdicts[b];
    if (v.choice != -1) return;
    const float temperature = p.temperatures ? p.temperatures[b] : 1.0f;
    const Draw d = draw_of(p, b, v, temperature);
    __shared__ double before[4];
    __shared__ int found[4], last[4];
    const double2* sums = p.sums + (int64_t)b * p.chunks;
    // every thread walks the chunks in order
    double total = 0.0;
    for (int c = 0; c < p.chunks; ++c) total += sums[c].x;
    const bool whole = !(total > 0.0);  // nothing is left of p: all of it
    if (whole) {
        total = 0.0;
        for (int c = 0; c < p.chunks; ++c) total += sums[c].y;
    }
    const double border = (double)p.uniforms[b * (p.drafts + 1) + p.drafts] * total;
    double running = 0.0, base = 0.0;
    int chunk = 0;
    for (int c = 0; c < p.chunks; ++c) {
        const double s = whole ? sums[c].y : sums[c].x;
        if (s > 0.0) {
            chunk = c;
            base = running;
            if (running + s > border) break;
        }
        running += s;
    }
    // this thread's run of 4 E indices in order
    double w[E][4], mine = 0.0;
    const int first = (chunk * kThreads + t) * E * 4;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        double rest[4], all[4];
        d.at(first + 4 * e, rest, all);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            w[e][c] = whole ? all[c] : rest[c];
            mine += w[e][c];
        }
    }
    double upto = mine;  // inclusive over the wave's lanes
    for (int m = 1; m < 64; m <<= 1) {
        const uint64_t u = (uint64_t)__double_as_longlong(upto);
        const uint32_t lo = (uint32_t)__shfl_up((int)(uint32_t)u, m), hi = (uint32_t)__shfl_up((int)(uint32_t)(u >> 32), m);
        if (lane >= m) upto += __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
    }
    if (lane == 63) before[wave] = upto;
    __syncthreads();
    double sum = base + (upto - mine);
    for (int k = 0; k < wave; ++k) sum += before[k];
    int hit = 0x7fffffff, most = -1;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (w[e][c] > 0.0) {
                sum += w[e][c];
                const int i = first + 4 * e + c;
                if (sum > border && hit == 0x7fffffff) hit = i;
                most = i;
            }
    for (int m = 1; m < 64; m <<= 1) {
        hit = min(hit, __shfl_xor(hit, m));
        most = max(most, __shfl_xor(most, m));
    }
    if (lane == 0) {
        found[wave] = hit;
        last[wave] = most;
    }
    __syncthreads();
    if (t == 0) {
        hit = min(min(found[0], found[1]), min(found[2], found[3]));
        // past the end by a rounding, or by a uniform of 1: the last index with a weight
        if (hit == 0x7fffffff) hit = max(max(last[0], last[1]), max(last[2], last[3]));
        const int at = b * (p.drafts + 1) + v.at;
        p.emitted[at] = hit;
        if (p.probabilities) p.probabilities[at] = (float)(weight(d.p_row[hit], v.p_peak, d.warm) * v.p_scale);
    }
}

struct VerifyPlan {
    int rows = 0, each = 1, chunks = 0;  // each: 4-logit loads a thread
    size_t sums_at = 0, verdicts_at = 0, bytes = 0;
};

VerifyPlan verify_plan(int sequences, int drafts, int vocab) {
    VerifyPlan n;
    n.rows = 2 * drafts + 1;
    // 16 logits a thread where that still gives the chip four blocks a CU, else 4
    n.each = (int64_t)sequences * n.rows * ((vocab + 4095) / 4096) >= 1024 ? 4 : 1;
    n.chunks = (vocab + 1024 * n.each - 1) / (1024 * n.each);
    n.sums_at = aligned_bytes((size_t)sequences * n.rows * n.chunks * sizeof(RowPart));
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
    p.chunks = n.chunks;
    hipStream_t s = (hipStream_t)stream;
    const dim3 rows(n.chunks, p.rows, sequences), run(n.chunks, sequences), draw(sequences), block(kThreads);
    if (n.each == 4) {
        rn_launch(verify_rows_kernel<4>, rows, block, 0, s, p);
        rn_launch(verify_run_kernel<4>, run, block, 0, s, p);
        rn_launch(verify_draw_kernel<4>, draw, block, 0, s, p);
    } else {
        rn_launch(verify_rows_kernel<1>, rows, block, 0, s, p);
        rn_launch(verify_run_kernel<1>, run, block, 0, s, p);
        rn_launch(verify_draw_kernel<1>, draw, block, 0, s, p);
    }
    SV_HIP(hipGetLastError());
    return RN_OK;
}
