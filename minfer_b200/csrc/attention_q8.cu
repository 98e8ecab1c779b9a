// Attention of a step's tokens over a paged cache of 8-bit keys and values (q8.cuh says what a vector's
// codes and scale are).  Row b brings tokens cu_seqlens[b] .. cu_seqlens[b+1]-1, at positions
// seq_end[b] - count .. seq_end[b] - 1; a token at p sees the positions j <= p (and, with a window,
// p - j < window), whose keys the pages hold, the step's own included:
//
//   o_i = sum_j p_ij vs_j vc_j / sum_j p_ij,   p_ij = exp(scale q_i . kc_j ks_j - max)
//
// kc, vc codes and ks, vs scales.  A key's scale goes on its score and a value's on its probability, so
// the codes are multiplied as they are.  A token that sees nothing gets zeros.
//
// All tokens of a row and all query heads of a key/value head share the keys: their rows are the rows of
// one matrix product, r = token * group + head.
#include "q8.cuh"

#include <cooperative_groups.h>

struct AttnQ8Args {
    const void* q;                 // [tokens][n_heads][hd]
    const uint8_t* k_codes;        // [pages][n_kv][64][hd]
    const uint8_t* v_codes;
    const float* k_scales;         // [pages][n_kv][64]
    const float* v_scales;
    const int* cu_seqlens;
    const int* seq_end;
    const int* page_table;
    int table_stride, ring, n_pages;
    void* out;                     // [tokens][n_heads][hd]
    float* partial;                // [tokens][n_heads][n_splits][hd + 2] where n_splits > 1
    int n_tokens, n_heads, n_kv, hd, window;
    int n_splits;                  // parts that a row's pages are shared out to
    int q_groups;                  // blocks along a row's matrix rows
    float scale;
    unsigned* status;
};

#define AQ_NEG (-INFINITY)
#define AQ_MAX_SPLITS 4096

__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void cp16(uint32_t to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ float ex2(float x) {            // 2^x; results below the normal range are 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
__device__ __forceinline__ float lds32(uint32_t at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}

// ------------------------------------------------------------------------------------------
// bfloat16 queries, head size 64 or 128, on the tensor cores (m16n8k16, halves into float32).
//
// Both products are transposed: scores S^T = K Q^T and outputs O^T = V^T P^T, so that keys (then dimensions)
// are the 16 rows of a tile and matrix rows its 8 columns.  A group of seven heads then wastes one column in
// eight, where as rows it would waste nine in sixteen, and a warp holds half the registers.
//
// A warp owns 16 keys of every page of its block's split (four warps, 64 positions a page) and streams
// them through a ring of its own in shared memory, filled by cp.async: no barrier between warps until
// the end, where the four results are joined.  An 8-bit code is an exact half, so both products run on
// halves: a query's row is brought to [2^14, 2^15) by a power of two first (a half has more mantissa
// than a bfloat16, and 2^-28 of a row's largest element is still exact), the power goes into the
// float32 factor of its scores.
//
// Values' scales differ from key to key, and a half holds 2^-14..2^16: so beside the reference m of its
// scores a row carries a reference w of its weights p_j vs_j, and what is rounded to halves is p_j vs_j / w
// (off by 2^-11, where a bfloat16 probability is off by 2^-8).  Both references are maxima of what came
// before, moved up (and outputs rescaled) only when a score passes m by more than 8 powers of two or a
// weight passes w by more than 10: nothing is near overflow until then, sums are float32, and the usual
// step needs one vote and no exchange between lanes.
//
// Layouts: row r of a score tile is key 4 (r' >> 1) + 2 (r >> 3) + (r & 1), r' = r & 7, of the step's 16, so that
// the keys a thread multiplies values of are the four from 4 t on.  Both operands of a score see the same
// order of dimensions (a thread takes 16 neighbouring codes of a key: one load feeds four k-steps); rows g and
// g + 8 of output tile j are dimensions (HD / 8) g + 2 j and + 1, so a thread ends up with HD / 8 neighbouring ones.
// ------------------------------------------------------------------------------------------
#define AQ_WARPS 4
#define AQ_KEYS 16
#define AQ_SCORE_ROOM 8.0f        // powers of two
#define AQ_WEIGHT_ROOM 1024.0f

template <int HD> struct AqTile {
    static constexpr int CPR = HD / 16;                    // 16-byte chunks a vector
    static constexpr int CODES = AQ_KEYS * HD;             // bytes of codes, K or V
    static constexpr int STAGE = 2 * CODES + 2 * AQ_KEYS * 4;
    // where chunk c of row r lies: K and V are permuted so that the eight lanes that a 128-bit access serves
    // at once (sixteen of a 64-bit one) meet different banks
    __device__ static __forceinline__ int k_at(int r, int c) {
        return (HD == 128 ? r * CPR + (c ^ ((r & 1) << 2)) : r * CPR + c) * 16;
    }
    __device__ static __forceinline__ int v_at(int r, int c) { return ((r * CPR + c) ^ (((r >> 2) & 3) << 1)) * 16; }
};

__device__ __forceinline__ uint32_t transposed(uint32_t x) {          // an 8 x 8 tile of halves
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float over_keys_max(float v) {             // over the eight lanes of one t
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

// NT: tiles of 8 matrix rows a block takes.  CLUSTER: the splits of a row are the blocks of a cluster, which
// join their results through distributed shared memory; else each leaves a partial result for
// attention_q8_merge_kernel.
template <int HD, int FMT, int NT, bool CLUSTER, int STAGES, int MINB>
__global__ void __launch_bounds__(AQ_WARPS * 32, MINB) attention_q8_mma_kernel(AttnQ8Args a) {
    using T = AqTile<HD>;
    namespace cg = cooperative_groups;
    constexpr int OT = HD / 16;                            // output tiles of 16 dimensions
    constexpr int OS = HD + 4;                             // floats a row of the joining buffer
    constexpr int ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t aq_smem[];
    __shared__ float ml_s[AQ_WARPS][ROWS][3];
    __shared__ float f_s[AQ_WARPS][ROWS];
    __shared__ float2 row_s[ROWS];                         // the block's maximum and sum of each row
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, hk = blockIdx.y / a.q_groups, qg = blockIdx.y - hk * a.q_groups, b = blockIdx.z;
    const int G = a.n_heads / a.n_kv;
    const int tok0 = a.cu_seqlens[b], count = a.cu_seqlens[b + 1] - tok0, end = a.seq_end[b];
    const int r0 = qg * ROWS, rows = min(ROWS, count * G - r0);           // the block's matrix rows
    // (uniform over a cluster)
    if (rows <= 0 || tok0 < 0 || tok0 + count > a.n_tokens) { pdl_wait(); return; }
    // what the block's queries see together: [lo, hi); and every one of them: [lo_in, hi_in)
    const int first = end - count + r0 / G, last = end - count + (r0 + rows - 1) / G;
    const int lo_all = a.window > 0 ? max(0, first - a.window + 1) : 0;
    const int lo_in = a.window > 0 ? max(0, last - a.window + 1) : 0, hi_in = first + 1;
    // the row's own pages, shared out evenly
    const int base0 = lo_all & ~(MF_PAGE - 1), pages = max(0, (last - base0 + MF_PAGE) / MF_PAGE);
    const int chunk = (pages + a.n_splits - 1) / a.n_splits * MF_PAGE;
    const int base = base0 + split * chunk;
    const int lo = max(lo_all, base), hi = min(last + 1, base + chunk);
    const int n_it = hi > lo ? (hi - base + MF_PAGE - 1) / MF_PAGE : 0;
    const int* table = a.page_table + (size_t)b * a.table_stride;

    // ---- the ring ----
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(aq_smem) + warp * STAGES * T::STAGE;
    int ids = -1;                              // lane i: the page of iteration (it & ~31) + i
    auto look_up = [&](int it) {               // the next 32 page numbers
        const int p = base + (it + lane) * MF_PAGE;
        const int index = (a.ring > 0 ? p % a.ring : p) >> 6;
        ids = it + lane < n_it && index < a.table_stride ? table[index] : -1;
        // a page that is not there: its keys are seen by nobody, and the caller is told
        if (it + lane < n_it && (ids < 0 || ids >= a.n_pages)) {
            ids = -1;
            if (warp == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
        }
    };
    look_up(0);
    pdl_wait();
    unsigned filled = 0;                       // bit it & 31: the iteration's stage holds keys
    uint32_t fetch_to = ring0;
    auto fetch = [&](int it) {
        if ((it & 31) == 0 && it > 0) look_up(it);
        const int page = __shfl_sync(0xffffffffu, ids, it & 31);
        const int k0 = base + it * MF_PAGE + warp * AQ_KEYS;
        const bool here = it < n_it && page >= 0 && k0 < hi && k0 + AQ_KEYS > lo;
        filled = (filled & ~(1u << (it & 31))) | ((here ? 1u : 0u) << (it & 31));
        if (here) {
            const long long at = ((long long)page * a.n_kv + hk) * MF_PAGE + warp * AQ_KEYS;
            const uint8_t* kp = a.k_codes + at * HD + lane * 16;
            const uint8_t* vp = a.v_codes + at * HD + lane * 16;
#pragma unroll
            for (int i = 0; i < AQ_KEYS * T::CPR / 32; ++i) {
                const int u = i * 32 + lane, r = u / T::CPR, c = u % T::CPR;
                cp16(fetch_to + T::k_at(r, c), kp + i * 512);
                cp16(fetch_to + T::CODES + T::v_at(r, c), vp + i * 512);
            }
            if (lane < 8)
                cp16(fetch_to + 2 * T::CODES + lane * 16, (lane < 4 ? a.k_scales : a.v_scales - 16) + at + lane * 4);
        }
        fetch_to = fetch_to == ring0 + (STAGES - 1) * T::STAGE ? ring0 : fetch_to + T::STAGE;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);

    // ---- queries: a thread loads a part of row g of each tile; it works on the scores of rows 2 t, 2 t + 1 ----
    uint32_t qb[NT][HD / 16][2];
    float c_q[NT][2];                          // scale log2(e) / the row's power of two
    int hi_q[NT][2], lo_q[NT][2];              // positions the row sees: [lo, hi)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = n * 8 + g;
        uint4 w[HD / 64][2];
        unsigned top = 0;
        if (r < rows) {
            const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
            const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + ((size_t)(tok0 + token) * a.n_heads + head) * HD;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) w[c][i] = *reinterpret_cast<const uint4*>(q + 64 * c + 16 * t + 8 * i);
        } else {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) w[c][0] = w[c][1] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x[4] = {w[c][i].x, w[c][i].y, w[c][i].z, w[c][i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) top = max(top, max(x[j] & 0x7fffu, (x[j] >> 16) & 0x7fffu));
            }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the power of two: 2^(14 - exponent), from the exponent field (0: a row of zeros or of numbers
        // below the normal range, which 2^100 brings up and which count as zero below 2^-124)
        const int field = (int)(top >> 7);
        const int power = field == 0 ? 100 : min(141 - field, 100);
        const float up = __int_as_float((power + 127) << 23), down = __int_as_float((127 - power) << 23);
        const float c_row = field == 255 ? __int_as_float(0x7fc00000) : a.scale * 1.4426950408889634f * down;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            c_q[n][i] = __shfl_sync(0xffffffffu, c_row, (2 * t + i) * 4);
            const int rq = n * 8 + 2 * t + i;
            hi_q[n][i] = rq < rows ? end - count + (r0 + rq) / G + 1 : 0;
            lo_q[n][i] = rq < rows && a.window > 0 ? max(0, hi_q[n][i] - a.window) : 0;
        }
#pragma unroll
        for (int c = 0; c < HD / 64; ++c)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t x[4] = {w[c][i].x, w[c][i].y, w[c][i].z, w[c][i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // a non-finite element makes its row's factor NaN; here it only has to stay finite
                    const float f0 = field == 255 ? 0.0f : __uint_as_float(x[j] << 16) * up;
                    const float f1 = field == 255 ? 0.0f : __uint_as_float(x[j] & 0xffff0000u) * up;
                    // elements 8 i + 2 j, + 1 of the thread's 16: k-step 2 i + j / 2, first or second pair
                    qb[n][4 * c + 2 * i + (j >> 1)][j & 1] = pack_half2(f0, f1);
                }
            }
    }

    // references: neg = -m (infinity before the first key), norm = w, inv = 1 / w
    float neg[NT][2], l_q[NT][2], norm[NT][2], inv[NT][2], o[NT][OT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) { neg[n][i] = INFINITY; l_q[n][i] = norm[n][i] = inv[n][i] = 0.0f; }
#pragma unroll
        for (int j = 0; j < OT; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
    }

    const int key_a = 4 * (g >> 1) + (g & 1);              // the thread's keys: this one and the one 2 behind
    uint32_t stage = ring0;
    for (int it = 0; it < n_it; ++it) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
        if ((filled >> (it & 31)) & 1u) {
            const int k0 = base + it * MF_PAGE + warp * AQ_KEYS;
            // ---- scores (two accumulators a tile: half as long a chain) ----
            float sc[NT][2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) sc[n][h][0] = sc[n][h][1] = sc[n][h][2] = sc[n][h][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                const uint4 ka = lds128(stage + T::k_at(key_a, 4 * c + t)), kb = lds128(stage + T::k_at(key_a + 2, 4 * c + t));
                const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = q8_prepare<FMT>(wa[j]), y = q8_prepare<FMT>(wb[j]);
                    const uint32_t af[4] = {q8_halves<FMT, false>(x), q8_halves<FMT, false>(y), q8_halves<FMT, true>(x),
                                            q8_halves<FMT, true>(y)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(sc[n][j & 1], af, qb[n][4 * c + j][0], qb[n][4 * c + j][1]);
                }
            }
            // values: HD / 8 dimensions of the keys 4 t .. 4 t + 3
            uint32_t vw[4][HD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (HD == 128) {
                    const uint4 x = lds128(stage + T::CODES + T::v_at(4 * t + i, g));
                    vw[i][0] = x.x; vw[i][1] = x.y; vw[i][2] = x.z; vw[i][3] = x.w;
                } else {
                    const uint2 x = lds64(stage + T::CODES + T::v_at(4 * t + i, g >> 1) + 8 * (g & 1));
                    vw[i][0] = x.x; vw[i][1] = x.y;
                }
            }
            const float ks[2] = {lds32(stage + 2 * T::CODES + key_a * 4), lds32(stage + 2 * T::CODES + key_a * 4 + 8)};
            const float vs[2] = {lds32(stage + 2 * T::CODES + 64 + key_a * 4), lds32(stage + 2 * T::CODES + 64 + key_a * 4 + 8)};
            const bool edge = k0 < max(lo_in, lo) || k0 + AQ_KEYS > min(hi_in, hi);       // uniform
            if (edge) {
                // codes of places that no query of the block sees are anybody's
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (k0 + 4 * t + i < lo || k0 + 4 * t + i >= hi) {
#pragma unroll
                        for (int h = 0; h < HD / 32; ++h) vw[i][h] = 0u;
                    }
            }
            // ---- weights ----
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float x[2][2], w[2][2];                    // [key][row]
                unsigned gone = 0;                         // bit 2 k + i: row i does not see key k
                if (edge)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int at = k0 + key_a + 2 * k;
                            if (at >= min(hi_q[n][i], hi) || at < max(lo_q[n][i], lo)) gone |= 1u << (2 * k + i);
                        }
                auto weigh = [&]() {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float s = sc[n][0][2 * k + i] + sc[n][1][2 * k + i];
                            x[k][i] = fmaf(s, c_q[n][i] * ks[k], neg[n][i]);
                            // (a key or value that is not seen may have any scale: NaN must not get in)
                            if (edge && ((gone >> (2 * k + i)) & 1u)) x[k][i] = AQ_NEG;
                            const float p = ex2(x[k][i]);
                            w[k][i] = p * (vs[k] * inv[n][i]);
                            if (edge && ((gone >> (2 * k + i)) & 1u)) w[k][i] = 0.0f;
                        }
                };
                weigh();
                const float most = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
                const float heaviest = fmaxf(fmaxf(w[0][0], w[0][1]), fmaxf(w[1][0], w[1][1]));
                if (__any_sync(0xffffffffu, most > AQ_SCORE_ROOM || heaviest > AQ_WEIGHT_ROOM)) {
                    // both references up to the maxima that are known now
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float s[2], top = AQ_NEG, big = 0.0f;
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            s[k] = (sc[n][0][2 * k + i] + sc[n][1][2 * k + i]) * (c_q[n][i] * ks[k]);
                            if ((gone >> (2 * k + i)) & 1u) s[k] = AQ_NEG;
                            top = fmaxf(top, s[k]);
                        }
                        const float before = -neg[n][i], m = fmaxf(before, over_keys_max(top));
                        const float f = before == AQ_NEG ? 0.0f : ex2(before - m);
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            if (!((gone >> (2 * k + i)) & 1u)) big = fmaxf(big, ex2(s[k] - m) * vs[k]);
                        const float held = norm[n][i] * f;
                        big = fmaxf(fmaxf(held, over_keys_max(big)), 7.5e-37f);            // (2^-120: 1 / w is finite)
                        neg[n][i] = -m;
                        l_q[n][i] *= f;
                        norm[n][i] = big;
                        inv[n][i] = __fdividef(1.0f, big);
                        const float down = held * inv[n][i];
#pragma unroll
                        for (int j = 0; j < OT; ++j) { o[n][j][i] *= down; o[n][j][2 + i] *= down; }
                    }
                    weigh();
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) l_q[n][i] += ex2(x[0][i]) + ex2(x[1][i]);
                pb[n][0] = transposed(pack_half2(w[0][0], w[0][1]));
                pb[n][1] = transposed(pack_half2(w[1][0], w[1][1]));
            }
            // ---- values: pairs of keys of one dimension ----
#pragma unroll
            for (int h = 0; h < HD / 32; ++h) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t x = q8_prepare<FMT>(__byte_perm(vw[0][h], vw[1][h], u ? 0x7362 : 0x5140));
                    const uint32_t y = q8_prepare<FMT>(__byte_perm(vw[2][h], vw[3][h], u ? 0x7362 : 0x5140));
                    const uint32_t af[4] = {q8_halves<FMT, false>(x), q8_halves<FMT, true>(x), q8_halves<FMT, false>(y),
                                            q8_halves<FMT, true>(y)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * h + u], af, pb[n][0], pb[n][1]);
                }
            }
        }
        __syncwarp();                          // the stage the next fetch fills was read an iteration ago
        fetch(it + STAGES - 1);
        stage = stage == ring0 + (STAGES - 1) * T::STAGE ? ring0 : stage + T::STAGE;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the four warps' results joined, in warp order ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float l = l_q[n][i];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            if (g == 0) {
                float* to = ml_s[warp][n * 8 + 2 * t + i];
                to[0] = -neg[n][i]; to[1] = l; to[2] = norm[n][i];
            }
        }
    __syncthreads();                           // also: every warp is done with its ring
    float* o_s = (float*)aq_smem;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float* row = o_s + ((size_t)warp * ROWS + n * 8 + 2 * t + i) * OS + (HD / 8) * g;
#pragma unroll
            for (int j = 0; j < OT; j += 2)
                *reinterpret_cast<float4*>(row + 2 * j) =
                    make_float4(o[n][j][i], o[n][j][2 + i], o[n][j + 1][i], o[n][j + 1][2 + i]);
        }
    if (tid < ROWS) {
        float m = AQ_NEG, l = 0.0f;
#pragma unroll
        for (int w = 0; w < AQ_WARPS; ++w) m = fmaxf(m, ml_s[w][tid][0]);
        const float m_use = m == AQ_NEG ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < AQ_WARPS; ++w) {
            const float f = exp2f(ml_s[w][tid][0] - m_use);
            f_s[w][tid] = f * ml_s[w][tid][2];
            l += ml_s[w][tid][1] * f;
        }
        row_s[tid] = make_float2(l != l ? INFINITY : m, l);      // NaN among the scores: joining must not pass over it
    }
    __syncthreads();
    // the block's row r, dimensions d .. d + 3, in units of its maximum
    auto joined = [&](int r, int d) -> float4 {
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < AQ_WARPS; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(o_s + ((size_t)w * ROWS + r) * OS + d);
            const float f = f_s[w][r];
            acc.x = fmaf(x.x, f, acc.x); acc.y = fmaf(x.y, f, acc.y);
            acc.z = fmaf(x.z, f, acc.z); acc.w = fmaf(x.w, f, acc.w);
        }
        return acc;
    };
    auto write_out = [&](int r, int d, float4 v, float by) {
        const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
        const __nv_bfloat162 x = __floats2bfloat162_rn(v.x * by, v.y * by);
        const __nv_bfloat162 y = __floats2bfloat162_rn(v.z * by, v.w * by);
        *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)(tok0 + token) * a.n_heads + head) * HD + d) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    };
    const int units = rows * (HD / 4);
    if constexpr (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        const int n = a.n_splits, rank = split;
        // the block's own sum over its warps goes where the first warp's was
        for (int i = tid; i < units; i += AQ_WARPS * 32) {
            const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
            *reinterpret_cast<float4*>(o_s + (size_t)r * OS + d) = joined(r, d);
        }
        cluster.sync();
        // every block writes its share of the rows' outputs
        for (int i = rank * AQ_WARPS * 32 + tid; i < units; i += n * AQ_WARPS * 32) {
            const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < n) {
                    ml[s] = *cluster.map_shared_rank(row_s + r, s);
                    x[s] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(o_s + (size_t)r * OS + d, s));
                }
            float m = AQ_NEG, l = 0.0f;
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < n) m = fmaxf(m, ml[s].x);
            const float m_use = m == AQ_NEG ? 0.0f : m;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < n) {
                    const float f = exp2f(ml[s].x - m_use);
                    l = fmaf(ml[s].y, f, l);
                    acc.x = fmaf(x[s].x, f, acc.x); acc.y = fmaf(x[s].y, f, acc.y);
                    acc.z = fmaf(x[s].z, f, acc.z); acc.w = fmaf(x[s].w, f, acc.w);
                }
            write_out(r, d, acc, l == 0.0f ? 0.0f : 1.0f / l);
        }
        cluster.sync();                        // nobody leaves while its memory is read
    } else if (a.n_splits > 1) {
        for (int r = tid; r < rows; r += AQ_WARPS * 32) {
            const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
            *reinterpret_cast<float2*>(a.partial + (((size_t)(tok0 + token) * a.n_heads + head) * a.n_splits + split) *
                                                       (HD + 2)) = row_s[r];
        }
        if (n_it == 0) return;                 // no key: the merge reads the maximum only
        for (int i = tid; i < units; i += AQ_WARPS * 32) {
            const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
            const float4 v = joined(r, d);
            const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
            float* p = a.partial + (((size_t)(tok0 + token) * a.n_heads + head) * a.n_splits + split) * (HD + 2) + 2 + d;
            *reinterpret_cast<float2*>(p) = make_float2(v.x, v.y);
            *reinterpret_cast<float2*>(p + 2) = make_float2(v.z, v.w);
        }
    } else {
        for (int i = tid; i < units; i += AQ_WARPS * 32) {
            const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
            const float l = row_s[r].y;
            write_out(r, d, joined(r, d), l == 0.0f ? 0.0f : 1.0f / l);
        }
    }
}

// ------------------------------------------------------------------------------------------
// Any head size that is a multiple of 16 up to 256, float32 or bfloat16 queries, in float32 on the
// FP32 pipe (the true 32-bit path).  A block takes up to eight matrix rows of one key/value head; 32
// keys at a time are turned into float32 codes in shared memory once for all of them, lanes are keys
// in the scores and dimensions in the sums.  Bound by the shared-memory reads of the products.
// ------------------------------------------------------------------------------------------
#define AG_WARPS 4
#define AG_ROWS 8
#define AG_KEYS 32

template <typename T, int FMT>
__global__ void __launch_bounds__(AG_WARPS * 32) attention_q8_generic_kernel(AttnQ8Args a) {
    extern __shared__ __align__(16) uint8_t ag_smem[];
    pdl_launch_dependents();
    const int hd = a.hd, hs = hd + 1;                      // odd rows: a column of keys meets every bank
    float* k_s = (float*)ag_smem;                          // [AG_KEYS][hs]
    float* v_s = k_s + AG_KEYS * hs;                       // [AG_KEYS][hd]
    float* q_s = v_s + AG_KEYS * hd;                       // [AG_ROWS][hd]
    float* ks_s = q_s + AG_ROWS * hd;                      // [AG_KEYS] each
    float* vs_s = ks_s + AG_KEYS;
    float* p_s = vs_s + AG_KEYS;                           // [AG_ROWS][AG_KEYS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.x, hk = blockIdx.y / a.q_groups, qg = blockIdx.y - hk * a.q_groups, b = blockIdx.z;
    const int G = a.n_heads / a.n_kv;
    const int tok0 = a.cu_seqlens[b], count = a.cu_seqlens[b + 1] - tok0, end = a.seq_end[b];
    const int r0 = qg * AG_ROWS, rows = min(AG_ROWS, count * G - r0);
    if (rows <= 0 || tok0 < 0 || tok0 + count > a.n_tokens) { pdl_wait(); return; }
    const int first = end - count + r0 / G, last = end - count + (r0 + rows - 1) / G;
    const int lo_all = a.window > 0 ? max(0, first - a.window + 1) : 0;
    const int base0 = lo_all & ~(MF_PAGE - 1), pages = max(0, (last - base0 + MF_PAGE) / MF_PAGE);
    const int chunk = (pages + a.n_splits - 1) / a.n_splits * MF_PAGE;
    const int base = base0 + split * chunk;
    const int lo = max(lo_all, base), hi = min(last + 1, base + chunk);
    const int* table = a.page_table + (size_t)b * a.table_stride;
    pdl_wait();
    for (int i = tid; i < rows * hd; i += AG_WARPS * 32) {
        const int r = i / hd, d = i - r * hd, token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
        q_s[i] = to_f32(((const T*)a.q)[((size_t)(tok0 + token) * a.n_heads + head) * hd + d]) * a.scale;
    }
    constexpr int RW = AG_ROWS / AG_WARPS;                 // rows a warp
    constexpr int ND = 256 / 32;
    float m_r[RW], l_r[RW], acc[RW][ND];
    int lo_w[RW], hi_w[RW];
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        m_r[i] = AQ_NEG; l_r[i] = 0.0f;
        const int r = warp * RW + i;
        hi_w[i] = r < rows ? end - count + (r0 + r) / G + 1 : 0;
        lo_w[i] = r < rows && a.window > 0 ? max(0, hi_w[i] - a.window) : 0;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[i][d] = 0.0f;
    }
    // steps of 32 positions from a page's border: a step lies in one page
    for (int j0 = lo & ~(AG_KEYS - 1); j0 < hi; j0 += AG_KEYS) {
        const int index = (a.ring > 0 ? j0 % a.ring : j0) >> 6;
        int page = index < a.table_stride ? table[index] : -1;
        if (page < 0 || page >= a.n_pages) {               // (uniform over the block)
            if (tid == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
            continue;
        }
        const long long at = ((long long)page * a.n_kv + hk) * MF_PAGE + (j0 & (MF_PAGE - 1));
        __syncthreads();                                   // the step before is done with the buffers
        for (int i = tid; i < 2 * AG_KEYS * hd / 16; i += AG_WARPS * 32) {
            const bool is_v = i >= AG_KEYS * hd / 16;
            const int u = is_v ? i - AG_KEYS * hd / 16 : i, r = u * 16 / hd, d = u * 16 - r * hd;
            uint4 w = *reinterpret_cast<const uint4*>((is_v ? a.v_codes : a.k_codes) + at * hd + u * 16);
            if (j0 + r < lo || j0 + r >= hi) w = make_uint4(0, 0, 0, 0);       // anybody's
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
            float* to = is_v ? v_s + r * hd + d : k_s + r * hs + d;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[4];
                q8_floats<FMT>(x[j], f);
#pragma unroll
                for (int e = 0; e < 4; ++e) to[4 * j + e] = f[e];
            }
        }
        if (tid < AG_KEYS) ks_s[tid] = a.k_scales[at + tid];
        else if (tid < 2 * AG_KEYS) vs_s[tid - AG_KEYS] = a.v_scales[at + tid - AG_KEYS];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const int r = warp * RW + i, j = j0 + lane;
            const bool seen = j >= max(lo_w[i], lo) && j < min(hi_w[i], hi);
            if (!__any_sync(0xffffffffu, seen)) continue;
            const float* kr = k_s + lane * hs;
            const float* qr = q_s + r * hd;
            float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
            for (int d = 0; d < hd; d += 4) {
                const float4 q4 = *reinterpret_cast<const float4*>(qr + d);
                s0 = fmaf(q4.x, kr[d], s0); s1 = fmaf(q4.y, kr[d + 1], s1);
                s2 = fmaf(q4.z, kr[d + 2], s2); s3 = fmaf(q4.w, kr[d + 3], s3);
            }
            const float s = seen ? ((s0 + s1) + (s2 + s3)) * ks_s[lane] : AQ_NEG;
            const float top = fmaxf(m_r[i], warp_max(s));
            const float m_use = top == AQ_NEG ? 0.0f : top;
            const float f = expf(m_r[i] - m_use), p = expf(s - m_use);
            l_r[i] = l_r[i] * f + warp_sum(p);
            m_r[i] = top;
            p_s[r * AG_KEYS + lane] = seen ? p * vs_s[lane] : 0.0f;
            __syncwarp();
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[i][d] *= f;
            for (int jj = 0; jj < AG_KEYS; ++jj) {
                const float w = p_s[r * AG_KEYS + jj];
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    if (lane + 32 * d < hd) acc[i][d] = fmaf(w, v_s[jj * hd + lane + 32 * d], acc[i][d]);
            }
            __syncwarp();
        }
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const int r = warp * RW + i;
        if (r >= rows) continue;
        const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
        const size_t th = (size_t)(tok0 + token) * a.n_heads + head;
        if (a.n_splits > 1) {
            float* p = a.partial + (th * a.n_splits + split) * (hd + 2);
            if (lane == 0) {
                // base-2 units, as the tensor-core kernel leaves them
                p[0] = l_r[i] != l_r[i] ? INFINITY : m_r[i] * 1.4426950408889634f;
                p[1] = l_r[i];
            }
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (lane + 32 * d < hd) p[2 + lane + 32 * d] = acc[i][d];
        } else {
            const float inv = l_r[i] == 0.0f ? 0.0f : 1.0f / l_r[i];
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (lane + 32 * d < hd) ((T*)a.out)[th * hd + lane + 32 * d] = from_f32<T>(acc[i][d] * inv);
        }
    }
}

// ------------------------------------------------------------------------------------------
// The splits of one (token, head) joined in split order.  Partial results: maximum (base 2), sum, then
// the unnormalised output; a split without a visible key has a maximum of -infinity and no output.
// ------------------------------------------------------------------------------------------
template <typename T>
__global__ void attention_q8_merge_kernel(const float* partial, T* __restrict__ out, int n_splits, int hd, int n_heads,
                                          const int* cu_seqlens, int n_rows) {
    pdl_prologue();
    extern __shared__ float mq_s[];                        // [n_splits] factors
    __shared__ float red_s[33];
    const size_t th = blockIdx.x;
    // tokens of no row stay as they are
    const int token = blockIdx.x / n_heads;
    if (token < cu_seqlens[0] || token >= cu_seqlens[n_rows]) return;
    const float* p = partial + th * n_splits * (hd + 2);
    float m = AQ_NEG;
    for (int s = threadIdx.x; s < n_splits; s += blockDim.x) m = fmaxf(m, p[(size_t)s * (hd + 2)]);
    m = block_max(m, red_s);
    const float m_use = m == AQ_NEG ? 0.0f : m;
    float l = 0.0f;
    for (int s = threadIdx.x; s < n_splits; s += blockDim.x) {
        const float ms = p[(size_t)s * (hd + 2)];
        const float f = exp2f(ms - m_use);                 // NaN for NaN's mark
        mq_s[s] = ms == AQ_NEG ? -1.0f : f;                // -1: no key, no output
        if (ms != AQ_NEG) l += p[(size_t)s * (hd + 2) + 1] * f;
    }
    l = block_sum(l, red_s);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int d = threadIdx.x; d < hd; d += blockDim.x) {
        float o = 0.0f;
#pragma unroll 8
        for (int s = 0; s < n_splits; ++s) {
            const float f = mq_s[s];
            if (f != -1.0f) o = fmaf(p[(size_t)s * (hd + 2) + 2 + d], f, o);
        }
        out[th * hd + d] = from_f32<T>(o * inv);
    }
}

// ---- host side ------------------------------------------------------------------------------
static bool aq_on_tensor_cores(int hd, int dtype) { return dtype == MF_DTYPE_BF16 && (hd == 64 || hd == 128); }

// matrix rows a block takes, from the most tokens a row brings
static int aq_block_rows(int max_row_tokens, int group, int hd, int dtype) {
    if (!aq_on_tensor_cores(hd, dtype)) return AG_ROWS;
    const long long tiles = ((long long)max_row_tokens * group + 7) / 8;
    if (tiles <= 4) return (int)tiles * 8;
    const long long blocks = (tiles + 3) / 4;
    return (int)((tiles + blocks - 1) / blocks) * 8;
}

#define AQ_CLUSTER 8                           // most splits that are joined in a cluster
// Into how many parts a row's keys are split.  `span`: the most positions the queries of one block can see,
// from a page's border on.
extern "C" int mf_attention_q8_plan(int n_rows, int max_row_tokens, int span, int n_heads, int n_kv, int hd, int dtype) {
    if (n_rows <= 0 || max_row_tokens <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return 1;
    const int br = aq_block_rows(max_row_tokens, n_heads / n_kv, hd, dtype);
    const long long groups = ((long long)max_row_tokens * (n_heads / n_kv) + br - 1) / br;
    const long long items = (long long)n_rows * n_kv * groups;
    const int pages = span <= 0 ? 1 : (span + MF_PAGE - 1) / MF_PAGE;
    static const int forced = getenv("AQ_SPLITS") ? atoi(getenv("AQ_SPLITS")) : 0;
    long long splits = forced ? forced : 3LL * mf_sm_count() / items;
    if (splits > (pages + 3) / 4) splits = (pages + 3) / 4;      // 256 keys a split at least
    if (splits > AQ_MAX_SPLITS) splits = AQ_MAX_SPLITS;
    if (splits < 1) splits = 1;
    if (aq_on_tensor_cores(hd, dtype) && splits <= 2 * AQ_CLUSTER) {
        int s = 1;
        while (2 * s <= splits && 2 * s <= AQ_CLUSTER) s *= 2;
        splits = s;
    }
    return (int)splits;
}

#define AQ_MAX_DEVICES 64
template <int HD, int FMT, int NT, bool CLUSTER, int STAGES, int MINB>
static int launch_mma_as(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    constexpr int ring = AQ_WARPS * STAGES * AqTile<HD>::STAGE, join = AQ_WARPS * 8 * NT * (HD + 4) * 4;
    constexpr int smem = ring > join ? ring : join;
    auto kernel = attention_q8_mma_kernel<HD, FMT, NT, CLUSTER, STAGES, MINB>;
    static bool opened[AQ_MAX_DEVICES] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= AQ_MAX_DEVICES || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return (int)e;
        if (dev >= 0 && dev < AQ_MAX_DEVICES) opened[dev] = true;
    }
    if (!CLUSTER) {
        mf_launch(kernel, grid, dim3(AQ_WARPS * 32), smem, stream, a);
        return MF_LAUNCH_CHECK();
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(AQ_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = grid.x; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = mf_pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, a);
    return MF_LAUNCH_CHECK();
}
template <int HD, int FMT, int NT, int STAGES, int MINB>
static int launch_mma(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    return a.n_splits > 1 && a.n_splits <= AQ_CLUSTER
               ? launch_mma_as<HD, FMT, NT, true, STAGES, MINB>(a, grid, stream)
               : launch_mma_as<HD, FMT, NT, false, STAGES, MINB>(a, grid, stream);
}
template <typename T, int FMT> static int launch_generic(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    const int smem = (AG_KEYS * (2 * a.hd + 1) + AG_ROWS * a.hd + 2 * AG_KEYS + AG_ROWS * AG_KEYS) * 4;
    constexpr int most = (AG_KEYS * (2 * 256 + 1) + AG_ROWS * 256 + 2 * AG_KEYS + AG_ROWS * AG_KEYS) * 4;
    static bool opened[AQ_MAX_DEVICES] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= AQ_MAX_DEVICES || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(attention_q8_generic_kernel<T, FMT>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, most))
            return (int)e;
        if (dev >= 0 && dev < AQ_MAX_DEVICES) opened[dev] = true;
    }
    mf_launch(attention_q8_generic_kernel<T, FMT>, grid, dim3(AG_WARPS * 32), smem, stream, a);
    return MF_LAUNCH_CHECK();
}

// Whether so many splits are joined by a second kernel, from partial results.
extern "C" int mf_attention_q8_merges(int n_splits, int hd, int dtype) {
    return n_splits > (aq_on_tensor_cores(hd, dtype) ? AQ_CLUSTER : 1);
}

// `n_splits`: any number from 1 on (mf_attention_q8_plan gives a good one); `partial` holds
// tokens * n_heads * n_splits * (hd + 2) floats where mf_attention_q8_merges says so.
extern "C" int mf_attention_q8(const void* q, const void* k_codes, const void* v_codes, const float* k_scales,
                               const float* v_scales, const int* cu_seqlens, const int* seq_end, const int* page_table,
                               int table_stride, int ring, int n_pages, void* out, float* partial, int n_tokens,
                               int n_rows, int max_row_tokens, int n_heads, int n_kv, int hd, int window, int n_splits,
                               float scale, int dtype, int fmt, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0 || n_rows <= 0 || max_row_tokens <= 0) return 0;
    if (hd % 16 != 0 || hd < 16 || hd > 256 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return MF_ERR_UNSUPPORTED;
    if ((dtype != MF_DTYPE_F32 && dtype != MF_DTYPE_BF16) || (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8))
        return MF_ERR_UNSUPPORTED;
    if (table_stride <= 0 || n_pages <= 0 || ring < 0 || ring % MF_PAGE != 0 || window < 0 || n_splits < 1 ||
        (partial == nullptr && mf_attention_q8_merges(n_splits, hd, dtype)) || status == nullptr)
        return MF_ERR_ARGUMENT;
    if (ring > 0 && (window <= 0 || max_row_tokens > ring - window + 1)) return MF_ERR_ARGUMENT;
    if (n_rows > 65535 || n_splits > AQ_MAX_SPLITS) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales |
         (uintptr_t)out) & 15)
        return MF_ERR_UNSUPPORTED;
    AttnQ8Args a{};
    a.q = q; a.k_codes = (const uint8_t*)k_codes; a.v_codes = (const uint8_t*)v_codes; a.k_scales = k_scales;
    a.v_scales = v_scales; a.cu_seqlens = cu_seqlens; a.seq_end = seq_end; a.page_table = page_table;
    a.table_stride = table_stride; a.ring = ring; a.n_pages = n_pages; a.out = out; a.partial = partial;
    a.n_tokens = n_tokens; a.n_heads = n_heads; a.n_kv = n_kv; a.hd = hd; a.window = window;
    a.n_splits = n_splits; a.scale = scale; a.status = status;
    const int G = n_heads / n_kv, br = aq_block_rows(max_row_tokens, G, hd, dtype);
    const long long groups = ((long long)max_row_tokens * G + br - 1) / br;
    if (groups * n_kv > 65535) return MF_ERR_UNSUPPORTED;
    a.q_groups = (int)groups;
    const dim3 grid(n_splits, (unsigned)(groups * n_kv), n_rows);
    int e;
    if (aq_on_tensor_cores(hd, dtype)) {
#define AQ_GO(HD, NT, STAGES, MINB)                                                      \
    (fmt == MF_Q8_E4M3 ? launch_mma<HD, MF_Q8_E4M3, NT, STAGES, MINB>(a, grid, stream)   \
                       : launch_mma<HD, MF_Q8_INT8, NT, STAGES, MINB>(a, grid, stream))
        if (hd == 128)
            e = br == 8 ? AQ_GO(128, 1, 4, 3) : br == 16 ? AQ_GO(128, 2, 4, 3) : br == 24 ? AQ_GO(128, 3, 4, 2) : AQ_GO(128, 4, 4, 2);
        else
            e = br == 8 ? AQ_GO(64, 1, 6, 4) : br == 16 ? AQ_GO(64, 2, 6, 4) : br == 24 ? AQ_GO(64, 3, 6, 4) : AQ_GO(64, 4, 6, 3);
#undef AQ_GO
    } else if (dtype == MF_DTYPE_F32) {
        e = fmt == MF_Q8_E4M3 ? launch_generic<float, MF_Q8_E4M3>(a, grid, stream)
                              : launch_generic<float, MF_Q8_INT8>(a, grid, stream);
    } else {
        e = fmt == MF_Q8_E4M3 ? launch_generic<__nv_bfloat16, MF_Q8_E4M3>(a, grid, stream)
                              : launch_generic<__nv_bfloat16, MF_Q8_INT8>(a, grid, stream);
    }
    if (e || !mf_attention_q8_merges(n_splits, hd, dtype)) return e;
    const int threads = hd >= 128 ? 128 : hd >= 64 ? 64 : 32;
    if ((long long)n_tokens * n_heads > 0x7fffffffLL) return MF_ERR_UNSUPPORTED;
    if (dtype == MF_DTYPE_F32)
        mf_launch(attention_q8_merge_kernel<float>, dim3((unsigned)(n_tokens * n_heads)), dim3(threads),
                  (size_t)n_splits * 4, stream, partial, (float*)out, n_splits, hd, n_heads, cu_seqlens, n_rows);
    else
        mf_launch(attention_q8_merge_kernel<__nv_bfloat16>, dim3((unsigned)(n_tokens * n_heads)), dim3(threads),
                  (size_t)n_splits * 4, stream, partial, (__nv_bfloat16*)out, n_splits, hd, n_heads, cu_seqlens, n_rows);
    return MF_LAUNCH_CHECK();
}
