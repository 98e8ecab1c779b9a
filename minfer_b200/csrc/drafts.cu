// Drafted tokens held against the target model's probabilities, from given random numbers.
//
// Sequence b brings n_b = cu[b+1] - cu[b] drafted tokens x_0 .. x_{n_b - 1} and n_b + 1 rows of logits, from
// row cu[b] + b on: row j is the target's distribution p_j of the token that x_j stands for, the last one
// that of the token behind all drafts.  With q_j the distribution that x_j was drawn from,
//
//   x_j is accepted while  u_j q_j(x_j) < p_j(x_j);
//   at the first j that is not, the sequence's token is drawn from max(0, p_j - q_j);
//   if all are accepted, from p_{n_b}:
//   the lowest index whose running sum exceeds r_b times the whole sum.
//
// p = softmax(logits / T).  q comes from logits of its own, or is 1 at x_j (a draft that was looked up, not
// drawn): then x_j is accepted with p_j(x_j) and the rest is p_j without x_j.  T below 1e-6: x_j is accepted
// if it is the row's first maximum, and the token is the first maximum of the row where that ends.
//
// A row that holds a NaN, or nothing above -infinity (or, for T > 0, +infinity), is no distribution: its draft
// is not accepted and the token is -1.
//
// Two launches.  The first reads every row once: the maximum and sum of a piece of 8,192 logits, which stay
// in registers between the two (bound by bytes).  The second joins the pieces, decides, and
// passes over the one row that the token comes from: a cluster of up to eight blocks a sequence, every warp a
// contiguous stretch of the vocabulary, whose sums all blocks see; the block whose stretch holds the answer has
// kept that stretch's sums in steps of 128 tokens, and goes through one step again (through the whole
// stretch, a step after the other: 25 us more).
//
// The token has to be the definition's: a running sum over 150,000 tokens has a border within 7e-6 of any
// number, and within 1e-8 of one number in 300.  So everything that a draw compares is double, the
// exponentials too (draft_exp); an acceptance turns on one border, and where no draw needs it a row's sum
// is one of float32 exponentials, kept in double.
#include "common.cuh"

#include <cooperative_groups.h>

#define DR_THREADS 256
#define DR_EACH 32                                   // logits a thread of the first launch holds
#define DR_PIECE (DR_THREADS * DR_EACH)
#define DR_CLUSTER 8                                 // most blocks a sequence
#define DR_WARPS 16
#define DR_STEPS 64                                  // most steps of a stretch
#define DR_KEPT 32                                   // places whose maximum and sum a block keeps

struct DraftArgs {
    const float* logits;                             // [n_drafts + n_seqs] rows
    const float* draft_logits;                       // [n_drafts] rows or null
    long long stride, draft_stride;
    const int* drafts;
    const int* cu;
    const float* accept_u;
    const float* draw_u;
    int* accepted;
    int* tokens;
    double2* pieces;                                 // [rows][n_pieces]: {maximum, sum}, or {key, NaN seen}
    int n_drafts, n_seqs, vocab, n_pieces;
    float inv_hi, inv_lo;                            // 1 / T = hi + lo (an error in it would tilt every weight)
    float temperature;
    int greedy;
};

// exp((logit - top) / T) in double to 2e-12 of the result, by the table-driven method (P. T. P. Tang, 1989):
// the exponent is (32 k + j + r) ln 2 / 32 with |r| <= 1/2, so the result is 2^k 2^(j/32) exp(r ln 2 / 32), the last
// factor its series up to the fourth power.  0 below exp(-690) and for -infinity; NaN stays NaN; +infinity
// against itself counts as nothing.  Ten operations in double, beside which the look-up and the exponent's
// bits are integer work.
#define DR_TABLE 32
struct DraftExp {
    double steps, off;                               // 32 / (T ln 2), and -top times that
    float least;                                     // logits up to here weigh nothing
};
__device__ __forceinline__ void draft_table(double* table) {
    if (threadIdx.x < DR_TABLE) table[threadIdx.x] = exp2((double)threadIdx.x / DR_TABLE);
}
__device__ __forceinline__ DraftExp draft_against(const DraftArgs& a, float top) {
    DraftExp e;
    e.steps = ((double)a.inv_hi + (double)a.inv_lo) * (DR_TABLE * 1.4426950408889634074);
    e.off = -(double)top * e.steps;
    e.least = top - 690.0f * a.temperature;
    return e;
}
__device__ __forceinline__ double draft_exp(float logit, const DraftExp& e, const double* table) {
    constexpr double L = 0.69314718055994530942 / DR_TABLE;
    const double x = fma((double)logit, e.steps, e.off);
    const double magic = 6755399441055744.0;                              // 1.5 2^52: the sum's low word is round(x)
    const double shifted = x + magic;
    const int n = __double2loint(shifted);
    const double r = x - (shifted - magic);
    double q = fma(r, L * L * L * L / 24.0, L * L * L / 6.0);
    q = fma(q, r, L * L / 2.0);
    q = fma(q, r, L);
    q = fma(q, r, 1.0);
    const double t = table[n & (DR_TABLE - 1)];
    const double scaled = __hiloint2double(__double2hiint(t) + ((n >> 5) << 20), __double2loint(t));
    return logit <= e.least ? 0.0 : q * scaled;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ float weight_of(float logit, float top, const DraftArgs& a) {
    // (infinity times a residue of 1 / T would be NaN; a NaN stays)
    const float apart = logit - top, d = apart < -1e30f ? -1e30f : apart;
    return expf(fmaf(d, a.inv_hi, d * a.inv_lo));
}
// larger values first, then lower indices; -0 and +0 are one value
__device__ __forceinline__ unsigned long long place_key(float v, int index) {
    unsigned u = __float_as_uint(v + 0.0f);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)u << 32) | (unsigned)(0x7fffffff - index);
}

// EXACT: the sums are what a draw compares with (target and draft distributions are subtracted)
template <bool VEC, bool EXACT>
__global__ void __launch_bounds__(DR_THREADS) draft_pieces_kernel(DraftArgs a) {
    __shared__ double table_s[DR_TABLE];
    if (EXACT) draft_table(table_s);
    pdl_prologue();
    __shared__ float red_s[33];
    __shared__ double sum_s[DR_THREADS / 32];
    __shared__ unsigned long long key_s[DR_THREADS / 32];
    const int row = blockIdx.x / a.n_pieces, piece = blockIdx.x - row * a.n_pieces;
    const int n_target = a.n_drafts + a.n_seqs;
    const float* x = row < n_target ? a.logits + (long long)row * a.stride
                                    : a.draft_logits + (long long)(row - n_target) * a.draft_stride;
    const int base = piece * DR_PIECE, tid = threadIdx.x;
    float v[DR_EACH];
    float top = -INFINITY;
    if (VEC) {
#pragma unroll
        for (int i = 0; i < DR_EACH / 4; ++i) {
            const int at = base + (i * DR_THREADS + tid) * 4;
            float4 w = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (at < a.vocab) w = *reinterpret_cast<const float4*>(x + at);      // (the vocabulary is a multiple of 4)
            v[4 * i] = w.x; v[4 * i + 1] = w.y; v[4 * i + 2] = w.z; v[4 * i + 3] = w.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < DR_EACH; ++i) {
            const int at = base + i * DR_THREADS + tid;
            v[i] = at < a.vocab ? x[at] : -INFINITY;
        }
    }
    if (a.greedy) {
        unsigned long long best = 0;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < DR_EACH; ++i) {
            const int at = VEC ? base + ((i >> 2) * DR_THREADS + tid) * 4 + (i & 3) : base + i * DR_THREADS + tid;
            bad |= v[i] != v[i];
            if (at < a.vocab && v[i] > -INFINITY) best = max(best, place_key(v[i], at));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if ((tid & 31) == 0) key_s[tid >> 5] = best;
        bad = __syncthreads_or(bad);
        if (tid == 0) {
            for (int w = 1; w < DR_THREADS / 32; ++w) best = max(best, key_s[w]);
            a.pieces[blockIdx.x] = make_double2(__longlong_as_double((long long)best), bad ? 1.0 : 0.0);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < DR_EACH; ++i) top = fmaxf(top, v[i]);
    top = block_max(top, red_s);
    const float m = top == -INFINITY ? 0.0f : top;   // (nothing but -infinity: a sum of 0)
    double sum = 0.0;
    if (EXACT) {
        const DraftExp e = draft_against(a, top);
        double part[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int i = 0; i < DR_EACH; ++i) part[i & 3] += draft_exp(v[i], e, table_s);
        sum = (part[0] + part[1]) + (part[2] + part[3]);
    } else {
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < DR_EACH; ++i) part[i & 3] += weight_of(v[i], m, a);
        sum = (double)(part[0] + part[1]) + (double)(part[2] + part[3]);
    }
    sum = warp_sum_d(sum);
    if ((tid & 31) == 0) sum_s[tid >> 5] = sum;
    __syncthreads();
    if (tid == 0) {
        double s = 0.0;
        for (int w = 0; w < DR_THREADS / 32; ++w) s += sum_s[w];
        a.pieces[blockIdx.x] = make_double2((double)top, s);
    }
}

// a row's maximum and sum from its pieces (every lane of the warp gets them; NaN: no distribution)
struct RowSum {
    double sum;
    float top;
};
__device__ __forceinline__ RowSum join_pieces(const DraftArgs& a, int row, const double* table) {
    const double2* p = a.pieces + (size_t)row * a.n_pieces;
    const int lane = threadIdx.x & 31;
    RowSum r;
    r.top = -INFINITY;
    double s = 0.0;
    // (32 pieces are 262,144 tokens: more only beyond that)
    for (int i0 = 0; i0 < a.n_pieces; i0 += 32) {
        const double2 v = i0 + lane < a.n_pieces ? p[i0 + lane] : make_double2((double)-INFINITY, 0.0);
        const float top = fmaxf(r.top, warp_max((float)v.x));
        const DraftExp e = draft_against(a, top);
        // (a piece of nothing but -infinity has a sum of 0, or NaN if that is among it: 0 times it)
        if (i0 > 0) s *= draft_exp(r.top, e, table);
        s += v.y * draft_exp((float)v.x, e, table);
        r.top = top;
    }
    s = warp_sum_d(s);
    r.sum = r.top > -INFINITY ? s : (double)NAN;
    return r;
}

// Of the warp's 128 weights (four neighbours a lane): the first one whose running sum, on top of `run`, lies
// beyond `want` (index -1: none does), and the last one that is above 0 (-1: none), each with the running
// sum in front of it.  `run` goes on by the sum.
struct Crossing {
    int first, last;
    double before_first, before_last;
};
__device__ __forceinline__ Crossing find_crossing(const double* w, double want, double* run) {
    const int lane = threadIdx.x & 31;
    const double sum = (w[0] + w[1]) + (w[2] + w[3]);
    double upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    double r = *run + (upto - sum), before_first = 0.0, before_last = 0.0;
    int first = -1, last = -1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double before = r;
        r += w[e];
        if (w[e] > 0.0) {
            last = 4 * lane + e; before_last = before;
            if (first < 0 && r > want) { first = last; before_first = before; }
        }
    }
    const unsigned hit = __ballot_sync(0xffffffffu, first >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
    const int from = hit ? __ffs(hit) - 1 : 0, at = any ? 31 - __clz(any) : 0;
    Crossing c;
    c.first = __shfl_sync(0xffffffffu, first, from);
    c.before_first = __shfl_sync(0xffffffffu, before_first, from);
    c.last = __shfl_sync(0xffffffffu, last, at);
    c.before_last = __shfl_sync(0xffffffffu, before_last, at);
    *run += __shfl_sync(0xffffffffu, upto, 31);
    return c;
}
// the sum of the cluster's stretches, the same in every warp
__device__ __forceinline__ double sum_of_stretches(const double* sums) {
    const int lane = threadIdx.x & 31;
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < DR_CLUSTER * DR_WARPS / 32; ++i) s += sums[lane * (DR_CLUSTER * DR_WARPS / 32) + i];
    return warp_sum_d(s);
}
static_assert(DR_CLUSTER * DR_WARPS == 128, "a lane takes four stretches");

// MINB: blocks an SM the registers are cut for (with one, four steps' loads and exponentials are in flight)
template <bool VEC, int MINB>
__global__ void __launch_bounds__(DR_WARPS * 32, MINB) draft_resolve_kernel(DraftArgs a, int blocks) {
    namespace cg = cooperative_groups;
    __shared__ double table_s[DR_TABLE];
    __shared__ double sums_s[2][DR_CLUSTER * DR_WARPS];      // the stretches' sums, of every warp of the cluster
    __shared__ double steps_s[DR_WARPS][DR_STEPS];           // this block's stretches, step by step
    __shared__ RowSum rows_s[DR_KEPT][2];                    // of the first places: target, draft
    __shared__ int stop_s;
    draft_table(table_s);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % blocks, b = blockIdx.x / blocks;
    if (tid < 2 * DR_CLUSTER * DR_WARPS) sums_s[0][tid] = 0.0;
    pdl_prologue();
    cg::cluster_group cluster = cg::this_cluster();
    const int d0 = a.cu[b], n = a.cu[b + 1] - d0;
    const bool fits = d0 >= 0 && n >= 0 && d0 + n <= a.n_drafts;       // (uniform over the cluster)
    const int row0 = d0 + b, n_target = a.n_drafts + a.n_seqs;
    if (!fits) {
        if (rank == 0 && tid == 0) { a.accepted[b] = 0; a.tokens[b] = -1; }
        return;
    }
    if (tid == 0) stop_s = n;
    __syncthreads();
    if (a.greedy) {
        if (rank != 0) return;                               // (no block of this cluster waits for another)
        // the first maximum of place j, -1 if there is none
        auto first_of = [&](int j) {
            const double2* p = a.pieces + (size_t)(row0 + j) * a.n_pieces;
            unsigned long long best = 0;
            bool bad = false;
            for (int i = lane; i < a.n_pieces; i += 32) {
                const double2 v = p[i];
                best = max(best, (unsigned long long)__double_as_longlong(v.x));
                bad |= v.y != 0.0;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            bad = __any_sync(0xffffffffu, bad) || best == 0;
            return bad ? -1 : 0x7fffffff - (int)(best & 0xffffffffu);
        };
        for (int j = warp; j < n; j += DR_WARPS) {
            const int first = first_of(j);
            if (lane == 0 && (first < 0 || first != a.drafts[d0 + j])) atomicMin(&stop_s, j);
        }
        __syncthreads();
        if (warp == 0) {
            const int first = first_of(stop_s);
            if (lane == 0) { a.accepted[b] = stop_s; a.tokens[b] = first; }
        }
        return;
    }
    // ---- which drafts are accepted (every block of the cluster finds the same) ----
    const bool with_q = a.draft_logits != nullptr;
    for (int j = warp; j <= n; j += DR_WARPS) {
        // (what does not wait for one another is asked for together)
        const int x = j < n ? a.drafts[d0 + j] : -1;
        const bool inside = x >= 0 && x < a.vocab;
        const float u = j < n ? a.accept_u[d0 + j] : 0.0f;
        const float at_p = inside ? a.logits[(long long)(row0 + j) * a.stride + x] : 0.0f;
        const float at_q = inside && with_q ? a.draft_logits[(long long)(d0 + j) * a.draft_stride + x] : 0.0f;
        // (both rows' sums side by side)
        const RowSum p = join_pieces(a, row0 + j, table_s);
        RowSum q{};
        if (j < n && with_q) q = join_pieces(a, n_target + d0 + j, table_s);
        if (lane == 0) {
            if (j < DR_KEPT) { rows_s[j][0] = p; rows_s[j][1] = q; }
            if (j < n) {
                const double px = draft_exp(at_p, draft_against(a, p.top), table_s) / p.sum;
                const double qx = with_q ? draft_exp(at_q, draft_against(a, q.top), table_s) / q.sum : 1.0;
                // (false for NaN, for a token outside the vocabulary, and for one that the target cannot give)
                if (!inside || !((double)u * qx < px)) atomicMin(&stop_s, j);
            }
        }
    }
    __syncthreads();
    const int stop = stop_s;
    bool less = stop < n;                                    // draw from what q leaves of p
    RowSum p, q;
    if (stop < DR_KEPT) {
        p = rows_s[stop][0]; q = rows_s[stop][1];
    } else {
        p = join_pieces(a, row0 + stop, table_s);
        q = RowSum{};
        if (less && with_q) q = join_pieces(a, n_target + d0 + stop, table_s);
    }
    if (!(p.sum > 0.0)) {                                    // no distribution (uniform over the cluster)
        if (rank == 0 && tid == 0) { a.accepted[b] = stop; a.tokens[b] = -1; }
        return;
    }
    // (weights in units of the target's sum: a draw only compares them with one another)
    const double ratio = less && with_q ? p.sum / q.sum : 0.0;
    const DraftExp of_p = draft_against(a, p.top), of_q = draft_against(a, q.top);
    const float* lp = a.logits + (long long)(row0 + stop) * a.stride;
    const float* lq = with_q ? a.draft_logits + (long long)(d0 + (less ? stop : 0)) * a.draft_stride : nullptr;
    const int x = less ? a.drafts[d0 + stop] : -1;
    // what token i weighs
    auto left = [&](int i, float vp, float vq) -> double {
        const double wp = draft_exp(vp, of_p, table_s);
        if (!less) return wp;
        if (!with_q) return i == x ? 0.0 : wp;
        return fmax(0.0, wp - draft_exp(vq, of_q, table_s) * ratio);      // (a NaN beside 0: 0)
    };
    // stretches are whole steps, a step `wide` times four neighbours a lane
    const int stretches = blocks * DR_WARPS;
    const int wide = (a.vocab + stretches * DR_STEPS * 128 - 1) / (stretches * DR_STEPS * 128), step = 128 * wide;
    const int n_steps = (a.vocab + stretches * step - 1) / (stretches * step);
    const int each = n_steps * step;
    // the four tokens of a lane from i0 on, as far as they are below the vocabulary
    auto four = [&](int i0, double* w) {
        float vp[4], vq[4];
        if (VEC && i0 + 3 < a.vocab) {
            const float4 v = *reinterpret_cast<const float4*>(lp + i0);
            vp[0] = v.x; vp[1] = v.y; vp[2] = v.z; vp[3] = v.w;
            if (less && with_q) {
                const float4 u = *reinterpret_cast<const float4*>(lq + i0);
                vq[0] = u.x; vq[1] = u.y; vq[2] = u.z; vq[3] = u.w;
            } else {
                vq[0] = vq[1] = vq[2] = vq[3] = 0.0f;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                vp[e] = i0 + e < a.vocab ? lp[i0 + e] : -INFINITY;
                vq[e] = i0 + e < a.vocab && less && with_q ? lq[i0 + e] : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = i0 + e < a.vocab ? left(i0 + e, vp[e], vq[e]) : 0.0;
    };
    cluster.sync();                                          // every block runs before another writes to it
    const int me = rank * DR_WARPS + warp, from = me * each;
    for (int round = 0; ; ++round) {
        double sum = 0.0;
        int s0 = 0;
        // four steps at a time where they lie inside the vocabulary: their loads and sums overlap
        if (VEC && wide == 1)
            for (; s0 + 4 <= n_steps && from + (s0 + 4) * 128 <= a.vocab; s0 += 4) {
                float4 vp[4], vq[4];
                double part[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i0 = from + (s0 + k) * 128 + 4 * lane;
                    vp[k] = *reinterpret_cast<const float4*>(lp + i0);
                    vq[k] = less && with_q ? *reinterpret_cast<const float4*>(lq + i0) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int i0 = from + (s0 + k) * 128 + 4 * lane;
                    part[k] = (left(i0, vp[k].x, vq[k].x) + left(i0 + 1, vp[k].y, vq[k].y)) +
                              (left(i0 + 2, vp[k].z, vq[k].z) + left(i0 + 3, vp[k].w, vq[k].w));
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                    for (int k = 0; k < 4; ++k) part[k] += __shfl_xor_sync(0xffffffffu, part[k], o);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (lane == 0) steps_s[warp][s0 + k] = part[k];
                    sum += part[k];
                }
            }
        for (int s = s0; s < n_steps; ++s) {
            double part = 0.0;
            for (int k = 0; k < wide; ++k) {
                const int i0 = from + s * step + k * 128;
                double w[4] = {0.0, 0.0, 0.0, 0.0};
                if (i0 < a.vocab) four(i0 + 4 * lane, w);
                part += (w[0] + w[1]) + (w[2] + w[3]);
            }
            part = warp_sum_d(part);
            if (lane == 0) steps_s[warp][s] = part;
            sum += part;
        }
        if (lane < blocks) *cluster.map_shared_rank(&sums_s[round][me], lane) = sum;
        cluster.sync();                                      // every block has every sum
        if (sum_of_stretches(sums_s[round]) > 0.0 || !less) break;
        // nothing is left of p (rounding, or a number of 1 or more): from p itself
        less = false;
    }
    // ---- the block whose stretch it is finds the token ----
    if (warp == 0) {
        const double* sums = sums_s[stop < n && !less ? 1 : 0];
        const double want = (double)a.draw_u[b] * sum_of_stretches(sums);
        // the stretch: the first whose end lies beyond `want`, else the last that holds anything
        double w[4], run = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = sums[4 * lane + e];
        const Crossing s = find_crossing(w, want, &run);
        const int pick = max(0, s.first >= 0 ? s.first : s.last);
        if (pick / DR_WARPS != rank) return;
        // the step of it, the same way, and the token of the step
        run = s.first >= 0 ? s.before_first : s.before_last;
        const double* parts = steps_s[pick % DR_WARPS];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = 4 * lane + e < n_steps ? parts[4 * lane + e] : 0.0;
        const Crossing t = find_crossing(w, want, &run);
        const int in = max(0, t.first >= 0 ? t.first : t.last);
        run = t.first >= 0 ? t.before_first : t.before_last;
        int token = -1, last = -1;
        for (int k = 0; k < wide && token < 0; ++k) {
            const int i0 = pick * each + in * step + k * 128;
            four(i0 + 4 * lane, w);
            const Crossing c = find_crossing(w, want, &run);
            if (c.first >= 0) token = i0 + c.first;
            if (c.last >= 0) last = i0 + c.last;
        }
        if (lane == 0) {
            a.accepted[b] = stop;
            a.tokens[b] = token >= 0 ? token : last;
        }
    }
}

template <bool VEC> static int drafts_launch(const DraftArgs& a, int rows, cudaStream_t stream) {
    const dim3 grid((unsigned)(rows * a.n_pieces));
    if (a.draft_logits != nullptr) mf_launch(draft_pieces_kernel<VEC, true>, grid, dim3(DR_THREADS), 0, stream, a);
    else mf_launch(draft_pieces_kernel<VEC, false>, grid, dim3(DR_THREADS), 0, stream, a);
    if (int e = MF_LAUNCH_CHECK()) return e;
    // as many blocks a sequence as the GPU holds at once: one an SM if that is the most a cluster takes, else two.
    // us, one / two an SM, both launches: 1 sequence of 4 drafts with their logits 21.4 / 23.3, 8 of 4 36.0 / 45.8, 64 of
    // 4 153 / 142, 64 of 0 to 7 looked up 78 / 70.
    int blocks = DR_CLUSTER;
    const bool few = (long long)a.n_seqs * blocks <= mf_sm_count();
    while (blocks > 1 && (long long)a.n_seqs * blocks > 2 * mf_sm_count()) blocks >>= 1;
    if (a.greedy) blocks = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.n_seqs * blocks);
    cfg.blockDim = dim3(DR_WARPS * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = mf_pdl_enabled() ? 2 : 1;
    if (few) cudaLaunchKernelEx(&cfg, draft_resolve_kernel<VEC, 1>, a, blocks);
    else cudaLaunchKernelEx(&cfg, draft_resolve_kernel<VEC, 2>, a, blocks);
    return MF_LAUNCH_CHECK();
}

// pieces a row of `vocab` logits is read in (the scratch holds 16 bytes for each)
extern "C" int mf_draft_pieces(int vocab) { return (vocab + DR_PIECE - 1) / DR_PIECE; }

extern "C" int mf_verify_drafts(const float* logits, long long stride, const int* drafts, const int* cu,
                                const float* draft_logits, long long draft_stride, const float* accept_u,
                                const float* draw_u, double temperature, int* accepted, int* tokens, void* pieces,
                                int n_drafts, int n_seqs, int vocab, cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (vocab <= 0 || n_drafts < 0 || !(temperature >= 0.0)) return MF_ERR_ARGUMENT;
    DraftArgs a{};
    a.logits = logits; a.stride = stride; a.drafts = drafts; a.cu = cu; a.draft_stride = draft_stride;
    a.accept_u = accept_u; a.draw_u = draw_u; a.accepted = accepted; a.tokens = tokens; a.pieces = (double2*)pieces;
    a.n_drafts = n_drafts; a.n_seqs = n_seqs; a.vocab = vocab; a.n_pieces = mf_draft_pieces(vocab);
    a.greedy = temperature < 1e-6;
    a.draft_logits = a.greedy || n_drafts == 0 ? nullptr : draft_logits;
    const double inv = a.greedy ? 0.0 : 1.0 / temperature;
    a.inv_hi = (float)inv;
    a.inv_lo = (float)(inv - (double)a.inv_hi);
    a.temperature = (float)temperature;
    const long long rows = (long long)n_drafts + n_seqs + (a.draft_logits ? n_drafts : 0);
    if (rows * a.n_pieces > 0x7fffffffLL || (long long)n_seqs * DR_CLUSTER > 0x7fffffffLL) return MF_ERR_UNSUPPORTED;
    const bool vec = vocab % 4 == 0 && stride % 4 == 0 && ((uintptr_t)logits & 15) == 0 &&
                     (a.draft_logits == nullptr || (draft_stride % 4 == 0 && ((uintptr_t)draft_logits & 15) == 0));
    return vec ? drafts_launch<true>(a, (int)rows, stream) : drafts_launch<false>(a, (int)rows, stream);
}
