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
// Three launches.  The first reads every row once: the maximum and sum of a piece of 8,192 logits, which stay
// in registers between the two.  The second joins the pieces, decides (every block of a sequence finds the
// same) and passes over the one row that the token comes from: a warp takes steps of 128 tokens and leaves
// their sums.  The third finds the step that holds the answer and goes through it again.  (The second and
// third as one, a cluster of eight blocks a sequence: 21 us for one sequence with four drafts over 151,936
// tokens where this takes 14, since eight SMs form 300,000 exponentials in double; 70 us for 64 of them
// where this takes 57.)  Of those 57 us the first launch is some 33, 5.9 TB/s of its 190 MB; the second forms
// ten million exponentials in double, twenty instructions each, and is bound by their latency and issue: 20 us
// with the 32 warps an SM that 64 registers leave room for and two steps in flight, 24 with 16 warps and four.
// Where the drafts have distributions of their own, all rows' exponentials are double: 129 us of 64 sequences.
// One sequence is bound by the latency of its three launches.
//
// The token has to be the definition's: a running sum over 150,000 tokens has a border within 7e-6 of any
// number, and within 1e-8 of one number in 300.  So everything that a draw compares is double, the
// exponentials too (draft_exp); an acceptance turns on one border, and where no draw needs it a row's sum
// is one of float32 exponentials, kept in double.
#include "common.cuh"

#define DR_THREADS 256
#define DR_EACH 32                                   // logits a thread of the first launch holds
#define DR_PIECE (DR_THREADS * DR_EACH)
#define DR_WARPS 8                                   // of the second launch's blocks
#define DR_HELD 4                                    // of those an SM holds at once
#define DR_MOST 128                                  // most of them a sequence
#define DR_AHEAD 2                                   // steps that a warp has in flight
#define DR_STEP 128                                  // tokens of a step: four neighbours a lane
#define DR_KEPT 32                                   // places whose maximum and sum a block keeps
#define DR_PICK 512                                  // threads of the third launch's blocks

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
    double* sums;                                    // [n_seqs][n_steps] of the row that the token comes from
    struct DraftCase* cases;                         // [n_seqs]
    int n_steps;
    int n_drafts, n_seqs, vocab, n_pieces;
    double base2;                                    // log2(e) / T
    float base2_hi, base2_lo;                        // their sum is that (an error in it would tilt every weight)
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
    e.steps = a.base2 * DR_TABLE;
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
    // (infinity times a residue would be NaN, so what is far below is brought near; a NaN stays)
    float d, w;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(logit - top), "f"(-3e38f));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaf(d, a.base2_hi, d * a.base2_lo)));
    return w;
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
// What the second launch has decided about a sequence, for the third.
struct DraftCase {
    double ratio;                                    // the target's sum over the draft's, where that is taken off
    float top_p, top_q;
    int stop;                                        // drafts accepted; -1: nothing is left to do
    int less;                                        // draw from what q leaves of p
};

// The weights of the row that a token comes from, in units of the target's sum (a draw only compares
// them with one another).
struct DraftRow {
    const float *lp, *lq;
    DraftExp of_p, of_q;
    double ratio;
    int x, vocab;
    __device__ __forceinline__ DraftRow(const DraftArgs& a, int b, int d0, const DraftCase& c) {
        const bool less = c.less != 0, with_q = a.draft_logits != nullptr;
        lp = a.logits + (long long)(d0 + b + c.stop) * a.stride;
        lq = less && with_q ? a.draft_logits + (long long)(d0 + c.stop) * a.draft_stride : nullptr;
        of_p = draft_against(a, c.top_p);
        of_q = draft_against(a, c.top_q);
        ratio = c.ratio;
        x = less && !with_q ? a.drafts[d0 + c.stop] : -1;
        vocab = a.vocab;
    }
    // the weights of a lane's four tokens from i0 on (a NaN that q brings: 0)
    __device__ __forceinline__ void weights(int i0, const float* vp, const float* vq, const double* table,
                                            double* w) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = draft_exp(vp[e], of_p, table);
        if (lq != nullptr) {
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = fmax(0.0, w[e] - draft_exp(vq[e], of_q, table) * ratio);
        } else if (x >= i0 && x < i0 + 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i0 + e == x) w[e] = 0.0;
        }
    }
    __device__ __forceinline__ double weight(int i0, const float* vp, const float* vq, const double* table) const {
        double w[4];
        weights(i0, vp, vq, table, w);
        return (w[0] + w[1]) + (w[2] + w[3]);
    }
    // a lane's four tokens from i0 on, as far as they are in the vocabulary
    template <bool VEC> __device__ __forceinline__ void load(int i0, float* vp, float* vq) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) vp[e] = vq[e] = -INFINITY;
        if (VEC) {                                   // (a multiple of 4 tokens)
            if (i0 < vocab) {
                const float4 v = *reinterpret_cast<const float4*>(lp + i0);
                vp[0] = v.x; vp[1] = v.y; vp[2] = v.z; vp[3] = v.w;
                if (lq != nullptr) {
                    const float4 u = *reinterpret_cast<const float4*>(lq + i0);
                    vq[0] = u.x; vq[1] = u.y; vq[2] = u.z; vq[3] = u.w;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i0 + e < vocab) {
                    vp[e] = lp[i0 + e];
                    if (lq != nullptr) vq[e] = lq[i0 + e];
                }
        }
    }
};

template <bool VEC>
__global__ void __launch_bounds__(DR_WARPS * 32, DR_HELD) draft_sums_kernel(DraftArgs a, int blocks) {
    __shared__ double table_s[DR_TABLE];
    __shared__ RowSum rows_s[DR_KEPT][2];                    // of the first places: target, draft
    __shared__ int stop_s;
    draft_table(table_s);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x % blocks, b = blockIdx.x / blocks;
    pdl_prologue();
    const int d0 = a.cu[b], end = a.cu[b + 1];
    // the sequence is done: so many drafts, this token
    auto answer = [&](int accepted, int token) {
        if (rank == 0 && tid == 0) {
            a.accepted[b] = accepted;
            a.tokens[b] = token;
            a.cases[b].stop = -1;
        }
    };
    if (d0 < 0 || end < d0 || end > a.n_drafts) { answer(0, -1); return; }
    const int n = end - d0, row0 = d0 + b, n_target = a.n_drafts + a.n_seqs;
    if (tid == 0) stop_s = n;
    __syncthreads();
    if (a.greedy) {
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
        if (warp == 0) answer(stop_s, first_of(stop_s));
        return;
    }
    // ---- which drafts are accepted ----
    const bool with_q = a.draft_logits != nullptr;
    for (int j = warp; j <= n; j += DR_WARPS) {
        // (what does not wait for one another is asked for together)
        const int x = j < n ? a.drafts[d0 + j] : -1;
        const bool inside = x >= 0 && x < a.vocab;
        const float u = j < n ? a.accept_u[d0 + j] : 0.0f;
        const float at_p = inside ? a.logits[(long long)(row0 + j) * a.stride + x] : 0.0f;
        const float at_q = inside && with_q ? a.draft_logits[(long long)(d0 + j) * a.draft_stride + x] : 0.0f;
        const RowSum p = join_pieces(a, row0 + j, table_s);
        RowSum q{};
        if (j < n && with_q) q = join_pieces(a, n_target + d0 + j, table_s);
        if (lane == 0) {
            if (j < DR_KEPT) { rows_s[j][0] = p; rows_s[j][1] = q; }
            if (j < n) {
                // u q(x) < p(x), the two sums multiplied out (false for NaN, for a token outside the
                // vocabulary, and for one that the target cannot give)
                const double ep = draft_exp(at_p, draft_against(a, p.top), table_s);
                const double eq = with_q ? draft_exp(at_q, draft_against(a, q.top), table_s) : 1.0;
                if (!inside || !((double)u * eq * p.sum < ep * (with_q ? q.sum : 1.0))) atomicMin(&stop_s, j);
            }
        }
    }
    __syncthreads();
    const int stop = stop_s;
    DraftCase c;
    c.stop = stop;
    c.less = stop < n;
    RowSum p, q;
    if (stop < DR_KEPT) {
        p = rows_s[stop][0]; q = rows_s[stop][1];
    } else {
        p = join_pieces(a, row0 + stop, table_s);
        q = RowSum{};
        if (c.less && with_q) q = join_pieces(a, n_target + d0 + stop, table_s);
    }
    if (!(p.sum > 0.0)) { answer(stop, -1); return; }        // no distribution
    c.ratio = c.less && with_q ? p.sum / q.sum : 0.0;
    c.top_p = p.top;
    c.top_q = q.top;
    if (rank == 0 && tid == 0) a.cases[b] = c;
    // ---- its sums, step by step; four steps of a warp at a time: their loads and exponentials overlap ----
    const DraftRow row(a, b, d0, c);
    double* sums = a.sums + (size_t)b * a.n_steps;
    const int warps = blocks * DR_WARPS;
    for (int s0 = rank * DR_WARPS + warp; s0 < a.n_steps; s0 += DR_AHEAD * warps) {
        float vp[DR_AHEAD][4], vq[DR_AHEAD][4];
        double part[DR_AHEAD];
#pragma unroll
        for (int k = 0; k < DR_AHEAD; ++k) {
            const int s = s0 + k * warps;
            row.template load<VEC>(s < a.n_steps ? s * DR_STEP + 4 * lane : 0x7ffffff0, vp[k], vq[k]);
        }
#pragma unroll
        for (int k = 0; k < DR_AHEAD; ++k) {
            const int i0 = (s0 + k * warps) * DR_STEP + 4 * lane;
            part[k] = 0.0;
            if (s0 + k * warps < a.n_steps)                  // (uniform over the warp)
                part[k] = row.weight(i0, vp[k], vq[k], table_s);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int k = 0; k < DR_AHEAD; ++k) part[k] += __shfl_xor_sync(0xffffffffu, part[k], o);
#pragma unroll
        for (int k = 0; k < DR_AHEAD; ++k)
            if (lane == 0 && s0 + k * warps < a.n_steps) sums[s0 + k * warps] = part[k];
    }
}

template <bool VEC>
__global__ void __launch_bounds__(DR_PICK) draft_pick_kernel(DraftArgs a) {
    __shared__ double table_s[DR_TABLE];
    __shared__ double ends_s[DR_PICK / 32];                  // the warps' sums
    draft_table(table_s);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
    pdl_prologue();
    DraftCase c = a.cases[b];
    if (c.stop < 0) return;
    const int d0 = a.cu[b];
    double* sums = a.sums + (size_t)b * a.n_steps;
    const double u = (double)a.draw_u[b];
    // a warp takes a stretch of whole chunks of 128 steps
    const int chunks = (a.n_steps + 127) / 128, each = (chunks + DR_PICK / 32 - 1) / (DR_PICK / 32) * 128;
    const int from = warp * each, to = min(a.n_steps, from + each);
    for (;;) {
        double mine = 0.0;
        for (int s = from + lane; s < to; s += 32) mine += sums[s];
        mine = warp_sum_d(mine);
        if (lane == 0) ends_s[warp] = mine;
        __syncthreads();
        double total = 0.0;
#pragma unroll
        for (int w = 0; w < DR_PICK / 32; ++w) total += ends_s[w];
        if (total > 0.0 || !c.less) break;                   // (uniform over the block)
        // nothing is left of p (rounding, or a number of 1 or more): from p itself
        c.less = 0;
        const DraftRow row(a, b, d0, c);
        for (int s = warp; s < a.n_steps; s += DR_PICK / 32) {
            float vp[4], vq[4];
            row.template load<VEC>(s * DR_STEP + 4 * lane, vp, vq);
            const double part = warp_sum_d(row.weight(s * DR_STEP + 4 * lane, vp, vq, table_s));
            if (lane == 0) sums[s] = part;
        }
        __syncthreads();
    }
    if (warp != 0) return;
    // the warp's stretch, then its chunk, then the step, then the token: each the first whose end lies beyond
    // `want`, else the last that holds anything
    double w[4], run = 0.0, want = 0.0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        w[e] = 4 * lane + e < DR_PICK / 32 ? ends_s[(4 * lane + e) % (DR_PICK / 32)] : 0.0;
        want += w[e];
    }
    want = u * warp_sum_d(want);
    const Crossing t = find_crossing(w, want, &run);
    const int at = max(0, t.first >= 0 ? t.first : t.last);
    run = t.first >= 0 ? t.before_first : t.before_last;
    int step = -1, last_step = 0;
    double before = 0.0, before_last = 0.0;
    for (int s0 = at * each; s0 < min(a.n_steps, (at + 1) * each) && step < 0; s0 += 128) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = s0 + 4 * lane + e < a.n_steps ? sums[s0 + 4 * lane + e] : 0.0;
        const Crossing k = find_crossing(w, want, &run);
        if (k.first >= 0) { step = s0 + k.first; before = k.before_first; }
        if (k.last >= 0) { last_step = s0 + k.last; before_last = k.before_last; }
    }
    if (step < 0) { step = last_step; before = before_last; }
    run = before;
    const DraftRow row(a, b, d0, c);
    float vp[4], vq[4];
    row.template load<VEC>(step * DR_STEP + 4 * lane, vp, vq);
    row.weights(step * DR_STEP + 4 * lane, vp, vq, table_s, w);
    const Crossing k = find_crossing(w, want, &run);
    if (lane == 0) {
        a.accepted[b] = c.stop;
        a.tokens[b] = step * DR_STEP + (k.first >= 0 ? k.first : k.last);
    }
}

template <bool VEC> static int drafts_launch(const DraftArgs& a, int rows, cudaStream_t stream) {
    const dim3 grid((unsigned)(rows * a.n_pieces));
    if (a.draft_logits != nullptr) mf_launch(draft_pieces_kernel<VEC, true>, grid, dim3(DR_THREADS), 0, stream, a);
    else mf_launch(draft_pieces_kernel<VEC, false>, grid, dim3(DR_THREADS), 0, stream, a);
    if (int e = MF_LAUNCH_CHECK()) return e;
    // what the GPU holds at once, and at least a step a warp
    int blocks = 1;
    if (!a.greedy) {
        blocks = min(DR_MOST, DR_HELD * mf_sm_count() / a.n_seqs);
        blocks = max(1, min(blocks, a.n_steps / DR_WARPS));
    }
    mf_launch(draft_sums_kernel<VEC>, dim3(a.n_seqs * blocks), dim3(DR_WARPS * 32), 0, stream, a, blocks);
    if (int e = MF_LAUNCH_CHECK()) return e;
    if (a.greedy) return 0;
    mf_launch(draft_pick_kernel<VEC>, dim3(a.n_seqs), dim3(DR_PICK), 0, stream, a);
    return MF_LAUNCH_CHECK();
}

static int draft_pieces(int vocab) { return (vocab + DR_PIECE - 1) / DR_PIECE; }
static int draft_steps_of(int vocab) { return (vocab + DR_STEP - 1) / DR_STEP; }
// The scratch of a call in bytes (16-byte aligned): `rows` of logits in all, drafts' among them.
extern "C" long long mf_draft_scratch(long long rows, int n_seqs, int vocab) {
    return rows * draft_pieces(vocab) * (long long)sizeof(double2) + (long long)n_seqs * (long long)sizeof(DraftCase) +
           (long long)n_seqs * draft_steps_of(vocab) * (long long)sizeof(double);
}

extern "C" int mf_verify_drafts(const float* logits, long long stride, const int* drafts, const int* cu,
                                const float* draft_logits, long long draft_stride, const float* accept_u,
                                const float* draw_u, double temperature, int* accepted, int* tokens, void* scratch,
                                int n_drafts, int n_seqs, int vocab, cudaStream_t stream) {
    if (n_seqs <= 0) return 0;
    if (vocab <= 0 || n_drafts < 0 || !(temperature >= 0.0 && temperature <= 1e30)) return MF_ERR_ARGUMENT;
    DraftArgs a{};
    a.logits = logits; a.stride = stride; a.drafts = drafts; a.cu = cu; a.draft_stride = draft_stride;
    a.accept_u = accept_u; a.draw_u = draw_u; a.accepted = accepted; a.tokens = tokens;
    a.n_drafts = n_drafts; a.n_seqs = n_seqs; a.vocab = vocab; a.n_pieces = draft_pieces(vocab);
    a.greedy = temperature < 1e-6;
    a.draft_logits = a.greedy || n_drafts == 0 ? nullptr : draft_logits;
    a.base2 = a.greedy ? 0.0 : 1.4426950408889634074 / temperature;
    a.base2_hi = (float)a.base2;
    a.base2_lo = (float)(a.base2 - (double)a.base2_hi);
    a.temperature = (float)temperature;
    const long long rows = (long long)n_drafts + n_seqs + (a.draft_logits ? n_drafts : 0);
    if (rows * a.n_pieces > 0x7fffffffLL || vocab > 0x7fffff00) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)scratch & 15) || scratch == nullptr) return MF_ERR_ARGUMENT;
    a.n_steps = draft_steps_of(vocab);
    a.pieces = (double2*)scratch;
    a.cases = (DraftCase*)(a.pieces + rows * a.n_pieces);
    a.sums = (double*)(a.cases + n_seqs);
    const bool vec = vocab % 4 == 0 && stride % 4 == 0 && ((uintptr_t)logits & 15) == 0 &&
                     (a.draft_logits == nullptr || (draft_stride % 4 == 0 && ((uintptr_t)draft_logits & 15) == 0));
    return vec ? drafts_launch<true>(a, (int)rows, stream) : drafts_launch<false>(a, (int)rows, stream);
}
