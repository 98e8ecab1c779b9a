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

#include <cmath>

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
    int chunk, n_splits;           // keys of a split (a multiple of 64)
    int q_groups;                  // blocks along a row's matrix rows
    float scale;
    unsigned* status;
};

#define AQ_NEG (-INFINITY)

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
// A warp owns 16 keys of every page of its block's split (four warps, 64 positions a page) and streams
// them through a ring of its own in shared memory, filled by cp.async: no barrier between warps until
// the end, where the four results are joined.  An 8-bit code is an exact half, so both products run on
// halves: a query's row is brought to [2^14, 2^15) by a power of two first (a half has more mantissa
// than a bfloat16, and 2^-28 of a row's largest element is still exact), the power goes into the
// float32 factor of its scores.
//
// Values' scales differ from key to key, and a half holds 2^-14..2^16: so beside the running maximum
// of its scores a row carries the largest weight so far, w = max_j p_j vs_j, and what is rounded to
// halves is p_j vs_j / w, at most 1 (off by 2^-11, where a bfloat16 probability is off by 2^-8).
// The output is kept in units of w: it is rescaled only when w grows against the scores' maximum.
//
// Layouts: column c of a score tile of 8 keys is key 4 (c & 1) + (c >> 1) of the tile, so that a
// thread's four columns of a 16-key step are keys t, t + 4, t + 8, t + 12: its value rows then lie in
// four different places of the banks.  Both operands of a score see the same order of dimensions (a
// thread takes 16 neighbouring codes of a key: one load feeds four k-steps); output column g of tile j
// is dimension (HD / 8) g + j, so a thread ends up with HD / 4 neighbouring dimensions.
// ------------------------------------------------------------------------------------------
#define AQ_WARPS 4
#define AQ_KEYS 16

template <int HD> struct AqTile {
    static constexpr int CPR = HD / 16;                    // 16-byte chunks a vector
    static constexpr int CODES = AQ_KEYS * HD;             // bytes of codes, K or V
    static constexpr int STAGE = 2 * CODES + 2 * AQ_KEYS * 4;
    // where chunk c of row r lies: K and V are permuted so that the eight lanes a 128-bit access serves
    // at once meet eight different groups of banks
    __device__ static __forceinline__ int k_at(int r, int c) {
        const int i = r * CPR + c;
        return (i ^ (((r >> 2) & 1) << 2)) * 16;
    }
    __device__ static __forceinline__ int v_at(int r, int c) {
        if (HD == 128) return (r * CPR + (c ^ ((r & 3) << 1))) * 16;
        return (r * CPR + (c ^ (((r >> 1) & 1) << 1))) * 16;
    }
};

template <int HD, int FMT, int MT, int STAGES, int MINB>
__global__ void __launch_bounds__(AQ_WARPS * 32, MINB) attention_q8_mma_kernel(AttnQ8Args a) {
    using T = AqTile<HD>;
    constexpr int OT = HD / 8;                             // output tiles of 8 columns
    constexpr int OS = HD + 8;                             // floats a row of the joining buffer
    extern __shared__ __align__(128) uint8_t aq_smem[];
    __shared__ float ml_s[AQ_WARPS][16 * MT][3];
    __shared__ float f_s[AQ_WARPS][16 * MT];
    __shared__ float sum_s[16 * MT];
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, hk = blockIdx.y / a.q_groups, qg = blockIdx.y - hk * a.q_groups, b = blockIdx.z;
    const int G = a.n_heads / a.n_kv;
    const int tok0 = a.cu_seqlens[b], count = a.cu_seqlens[b + 1] - tok0, end = a.seq_end[b];
    const int r0 = qg * 16 * MT, rows = min(16 * MT, count * G - r0);      // the block's matrix rows
    if (rows <= 0 || tok0 < 0 || tok0 + count > a.n_tokens) { pdl_wait(); return; }
    // what the block's queries see together: [lo, hi)
    const int first = end - count + r0 / G, last = end - count + (r0 + rows - 1) / G;
    const int lo_all = a.window > 0 ? max(0, first - a.window + 1) : 0;
    const int base = (lo_all & ~(MF_PAGE - 1)) + split * a.chunk;
    // (the last split takes whatever is left)
    const int lo = max(lo_all, base), hi = split == a.n_splits - 1 ? last + 1 : min(last + 1, base + a.chunk);
    const int n_it = hi > lo ? (hi - base + MF_PAGE - 1) / MF_PAGE : 0;
    const int* table = a.page_table + (size_t)b * a.table_stride;
    pdl_wait();

    // ---- queries ----
    uint32_t qa[MT][HD / 16][4];
    float c_r[MT][2];                          // scale log2(e) / the row's power of two, code unit included
    int hi_r[MT][2], lo_r[MT][2];              // positions the row sees: [lo, hi)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = m * 16 + g + 8 * e;
            uint4 w[HD / 64][2];
            unsigned top = 0;
            hi_r[m][e] = lo_r[m][e] = 0;
            if (r < rows) {
                const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
                const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + ((size_t)(tok0 + token) * a.n_heads + head) * HD;
                hi_r[m][e] = end - count + token + 1;
                lo_r[m][e] = a.window > 0 ? max(0, hi_r[m][e] - a.window) : 0;
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
            c_r[m][e] = field == 255 ? __int_as_float(0x7fc00000)
                                     : a.scale * 1.4426950408889634f * down * q8_half_unit<FMT>();
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
                        qa[m][4 * c + 2 * i + (j >> 1)][2 * (j & 1) + e] = pack_half2(f0, f1);
                    }
                }
        }
    }

    float m_r[MT][2], l_r[MT][2], w_r[MT][2], o[MT][OT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        m_r[m][0] = m_r[m][1] = AQ_NEG;
        l_r[m][0] = l_r[m][1] = w_r[m][0] = w_r[m][1] = 0.0f;
#pragma unroll
        for (int i = 0; i < OT; ++i) o[m][i][0] = o[m][i][1] = o[m][i][2] = o[m][i][3] = 0.0f;
    }

    // ---- the ring ----
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(aq_smem) + warp * STAGES * T::STAGE;
    int ids = -1;                              // lane i: the page of iteration (it & ~31) + i
    auto fetch = [&](int it) {
        if ((it & 31) == 0) {                  // the next 32 page numbers
            const int p = base + (it + lane) * MF_PAGE;
            const int index = (a.ring > 0 ? p % a.ring : p) >> 6;
            ids = it + lane < n_it && index < a.table_stride ? table[index] : -1;
            // a page that is not there: its keys are seen by nobody, and the caller is told
            if (it + lane < n_it && (ids < 0 || ids >= a.n_pages)) {
                ids = -1;
                if (warp == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
            }
        }
        const int page = __shfl_sync(0xffffffffu, ids, it & 31);
        const int k0 = base + it * MF_PAGE + warp * AQ_KEYS;
        if (it < n_it && page >= 0 && k0 < hi && k0 + AQ_KEYS > lo) {
            const long long at = ((long long)page * a.n_kv + hk) * MF_PAGE + warp * AQ_KEYS;
            const uint32_t to = ring0 + (it % STAGES) * T::STAGE;
            const uint8_t* kp = a.k_codes + at * HD;
            const uint8_t* vp = a.v_codes + at * HD;
#pragma unroll
            for (int i = 0; i < AQ_KEYS * T::CPR / 32; ++i) {
                const int u = i * 32 + lane, r = u / T::CPR, c = u - r * T::CPR;
                cp16(to + T::k_at(r, c), kp + u * 16);
                cp16(to + T::CODES + T::v_at(r, c), vp + u * 16);
            }
            if (lane < 8)
                cp16(to + 2 * T::CODES + lane * 16, (lane < 4 ? a.k_scales : a.v_scales - 16) + at + lane * 4);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        return page;
    };
    int page_of[STAGES];                       // whether an iteration's page is there
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) page_of[i] = fetch(i);

    for (int it0 = 0; it0 < n_it; it0 += STAGES) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) {
            const int it = it0 + s;
            if (it >= n_it) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncwarp();
            const int k0 = base + it * MF_PAGE + warp * AQ_KEYS;
            if (page_of[s] >= 0 && k0 < hi && k0 + AQ_KEYS > lo) {
                const uint32_t stage = ring0 + s * T::STAGE;
                // ---- scores ----
                float sc[MT][2][4];
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n) sc[m][n][0] = sc[m][n][1] = sc[m][n][2] = sc[m][n][3] = 0.0f;
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) {
                    uint4 kw[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n) kw[n] = lds128(stage + T::k_at(8 * n + 4 * (g & 1) + (g >> 1), 4 * c + t));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const uint32_t w = q8_prepare<FMT>(j == 0 ? kw[n].x : j == 1 ? kw[n].y : j == 2 ? kw[n].z : kw[n].w);
                            const uint32_t b0 = q8_halves<FMT, 0, 1>(w), b1 = q8_halves<FMT, 2, 3>(w);
#pragma unroll
                            for (int m = 0; m < MT; ++m) mma_f16(sc[m][n], qa[m][4 * c + j], b0, b1);
                        }
                }
                // ---- weights ----
                float ks[4], vs[4];            // keys t, t + 4, t + 8, t + 12
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ks[i] = lds32(stage + 2 * T::CODES + (4 * i + t) * 4);
                    vs[i] = lds32(stage + 2 * T::CODES + 64 + (4 * i + t) * 4);
                }
                uint32_t pa[MT][4];
#pragma unroll
                for (int m = 0; m < MT; ++m) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int h1 = hi_r[m][e] - k0 - t, l1 = lo_r[m][e] - k0 - t;
                        float x[4], w[4], top = m_r[m][e];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[i] = sc[m][i >> 1][2 * e + (i & 1)] * c_r[m][e] * ks[i];
                            if (4 * i >= h1 || 4 * i < l1) x[i] = AQ_NEG;
                            top = fmaxf(top, x[i]);
                        }
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        const float m_use = top == AQ_NEG ? 0.0f : top;
                        const float f = ex2(m_r[m][e] - m_use);                // 0 before the first key
                        m_r[m][e] = top;
                        l_r[m][e] *= f;
                        const float held = w_r[m][e] * f;                      // the largest weight so far
                        float big = held;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float p = ex2(x[i] - m_use);
                            l_r[m][e] += p;
                            // (a key that is not seen may have any scale: 0 * NaN must not get in)
                            w[i] = 4 * i >= h1 || 4 * i < l1 ? 0.0f : p * vs[i];
                            big = fmaxf(big, w[i]);
                        }
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
                        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
                        const float inv = big > 0.0f ? __fdividef(1.0f, big) : 0.0f;
                        w_r[m][e] = big;
                        if (__any_sync(0xffffffffu, big > held)) {
                            const float down = held * inv;
#pragma unroll
                            for (int i = 0; i < OT; ++i) { o[m][i][2 * e] *= down; o[m][i][2 * e + 1] *= down; }
                        }
                        pa[m][e] = pack_half2(w[0] * inv, w[1] * inv);
                        pa[m][2 + e] = pack_half2(w[2] * inv, w[3] * inv);
                    }
                }
                // ---- values ----
                const uint32_t vst = stage + T::CODES;
                uint32_t vw[4][HD / 32];       // HD / 8 dimensions of the rows t, t + 4, t + 8, t + 12
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (HD == 128) {
                        const uint4 x = lds128(vst + T::v_at(t + 4 * i, g));
                        vw[i][0] = x.x; vw[i][1] = x.y; vw[i][2] = x.z; vw[i][3] = x.w;
                    } else {
                        const uint2 x = lds64(vst + T::v_at(t + 4 * i, g >> 1) + 8 * (g & 1));
                        vw[i][0] = x.x; vw[i][1] = x.y;
                    }
                }
#pragma unroll
                for (int h = 0; h < HD / 32; ++h) {
                    const uint32_t w0 = q8_prepare<FMT>(vw[0][h]), w1 = q8_prepare<FMT>(vw[1][h]);
                    const uint32_t w2 = q8_prepare<FMT>(vw[2][h]), w3 = q8_prepare<FMT>(vw[3][h]);
                    const uint32_t lo4[4] = {q8_halves<FMT, 0, 4>(w0, w1), q8_halves<FMT, 1, 5>(w0, w1),
                                             q8_halves<FMT, 2, 6>(w0, w1), q8_halves<FMT, 3, 7>(w0, w1)};
                    const uint32_t hi4[4] = {q8_halves<FMT, 0, 4>(w2, w3), q8_halves<FMT, 1, 5>(w2, w3),
                                             q8_halves<FMT, 2, 6>(w2, w3), q8_halves<FMT, 3, 7>(w2, w3)};
#pragma unroll
                    for (int m = 0; m < MT; ++m)
#pragma unroll
                        for (int j = 0; j < 4; ++j) mma_f16(o[m][4 * h + j], pa[m], lo4[j], hi4[j]);
                }
            }
            __syncwarp();                      // the stage the next fetch fills was read an iteration ago
            page_of[(s + STAGES - 1) % STAGES] = fetch(it + STAGES - 1);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the four warps' results joined, in warp order ----
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l_r[m][e] += __shfl_xor_sync(0xffffffffu, l_r[m][e], 1);
            l_r[m][e] += __shfl_xor_sync(0xffffffffu, l_r[m][e], 2);
            if (t == 0) {
                ml_s[warp][m * 16 + g + 8 * e][0] = m_r[m][e];
                ml_s[warp][m * 16 + g + 8 * e][1] = l_r[m][e];
                ml_s[warp][m * 16 + g + 8 * e][2] = w_r[m][e];
            }
        }
    __syncthreads();                           // also: every warp is done with its ring
    float* o_s = (float*)aq_smem;
    if (tid < 16 * MT) {
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
        sum_s[tid] = l;
        if (tid < rows && a.n_splits > 1) {
            const int token = (r0 + tid) / G, head = hk * G + (r0 + tid) - token * G;
            float* p = a.partial + (((size_t)(tok0 + token) * a.n_heads + head) * a.n_splits + split) * (HD + 2);
            p[0] = l != l ? INFINITY : m;      // NaN among the scores: the merge must not pass over it
            p[1] = l;
        }
    }
    if (n_it == 0 && a.n_splits > 1) return;   // no key: the merge reads the maximum only
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        // dimensions (HD / 4) t .. of rows g and g + 8: the first half from a tile's column 2 t, the second from 2 t + 1
        float* row = o_s + ((size_t)warp * 16 * MT + m * 16 + g) * OS + (HD / 4) * t;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < OT; j += 4)
                    *reinterpret_cast<float4*>(row + (size_t)e * 8 * OS + h * OT + j) =
                        make_float4(o[m][j][2 * e + h], o[m][j + 1][2 * e + h], o[m][j + 2][2 * e + h], o[m][j + 3][2 * e + h]);
    }
    __syncthreads();
    for (int i = tid; i < rows * (HD / 4); i += AQ_WARPS * 32) {
        const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < AQ_WARPS; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(o_s + ((size_t)w * 16 * MT + r) * OS + d);
            const float f = f_s[w][r];
            acc[0] = fmaf(x.x, f, acc[0]); acc[1] = fmaf(x.y, f, acc[1]);
            acc[2] = fmaf(x.z, f, acc[2]); acc[3] = fmaf(x.w, f, acc[3]);
        }
        const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
        const size_t th = (size_t)(tok0 + token) * a.n_heads + head;
        if (a.n_splits > 1) {
            float* p = a.partial + (th * a.n_splits + split) * (HD + 2) + 2 + d;
#pragma unroll
            for (int e = 0; e < 4; e += 2)
                *reinterpret_cast<float2*>(p + e) =
                    make_float2(acc[e] * q8_half_unit<FMT>(), acc[e + 1] * q8_half_unit<FMT>());
        } else {
            const float l = sum_s[r], inv = l == 0.0f ? 0.0f : q8_half_unit<FMT>() / l;
            const __nv_bfloat162 x = __floats2bfloat162_rn(acc[0] * inv, acc[1] * inv);
            const __nv_bfloat162 y = __floats2bfloat162_rn(acc[2] * inv, acc[3] * inv);
            *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + th * HD + d) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
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
    const int base = (lo_all & ~(MF_PAGE - 1)) + split * a.chunk;
    // (the last split takes whatever is left)
    const int lo = max(lo_all, base), hi = split == a.n_splits - 1 ? last + 1 : min(last + 1, base + a.chunk);
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
            const uint4 w = *reinterpret_cast<const uint4*>((is_v ? a.v_codes : a.k_codes) + at * hd + u * 16);
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
    return (long long)max_row_tokens * group <= 16 ? 16 : 32;
}

// How the keys are split: (keys a split, splits).  `span`: the most positions the queries of one block
// can see, from a page's border on.
extern "C" int mf_attention_q8_plan(int n_rows, int max_row_tokens, int span, int n_heads, int n_kv, int hd, int dtype,
                                    int* chunk, int* n_splits) {
    if (n_rows <= 0 || max_row_tokens <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return MF_ERR_ARGUMENT;
    const int br = aq_block_rows(max_row_tokens, n_heads / n_kv, hd, dtype);
    const long long groups = ((long long)max_row_tokens * (n_heads / n_kv) + br - 1) / br;
    const long long items = (long long)n_rows * n_kv * groups;
    const long long want = 3LL * mf_sm_count();
    const int pages = span <= 0 ? 1 : (span + MF_PAGE - 1) / MF_PAGE;
    long long splits = want / items;
    if (splits < 1) splits = 1;
    // at least 256 keys a split
    if (splits > (pages + 3) / 4) splits = (pages + 3) / 4;
    const int per = (int)((pages + splits - 1) / splits);
    *chunk = per * MF_PAGE;
    *n_splits = (pages + per - 1) / per;
    return 0;
}

#define AQ_MAX_DEVICES 64
template <int HD, int FMT, int MT, int STAGES, int MINB>
static int launch_mma(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    constexpr int ring = AQ_WARPS * STAGES * AqTile<HD>::STAGE, join = AQ_WARPS * 16 * MT * (HD + 8) * 4;
    constexpr int smem = ring > join ? ring : join;
    static bool opened[AQ_MAX_DEVICES] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= AQ_MAX_DEVICES || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(attention_q8_mma_kernel<HD, FMT, MT, STAGES, MINB>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
            return (int)e;
        if (dev >= 0 && dev < AQ_MAX_DEVICES) opened[dev] = true;
    }
    mf_launch(attention_q8_mma_kernel<HD, FMT, MT, STAGES, MINB>, grid, dim3(AQ_WARPS * 32), smem, stream, a);
    return MF_LAUNCH_CHECK();
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

// `chunk` and `n_splits` from mf_attention_q8_plan for the same sizes; `partial` holds
// tokens * n_heads * n_splits * (hd + 2) floats where n_splits > 1.
extern "C" int mf_attention_q8(const void* q, const void* k_codes, const void* v_codes, const float* k_scales,
                               const float* v_scales, const int* cu_seqlens, const int* seq_end, const int* page_table,
                               int table_stride, int ring, int n_pages, void* out, float* partial, int n_tokens,
                               int n_rows, int max_row_tokens, int n_heads, int n_kv, int hd, int window, int chunk,
                               int n_splits, float scale, int dtype, int fmt, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0 || n_rows <= 0 || max_row_tokens <= 0) return 0;
    if (hd % 16 != 0 || hd < 16 || hd > 256 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return MF_ERR_UNSUPPORTED;
    if ((dtype != MF_DTYPE_F32 && dtype != MF_DTYPE_BF16) || (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8))
        return MF_ERR_UNSUPPORTED;
    if (table_stride <= 0 || n_pages <= 0 || ring < 0 || ring % MF_PAGE != 0 || window < 0 || chunk <= 0 ||
        chunk % MF_PAGE != 0 || n_splits < 1 || (n_splits > 1 && partial == nullptr) || status == nullptr)
        return MF_ERR_ARGUMENT;
    if (ring > 0 && (window <= 0 || max_row_tokens > ring - window + 1)) return MF_ERR_ARGUMENT;
    if (n_rows > 65535 || n_splits > 6000) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales |
         (uintptr_t)out) & 15)
        return MF_ERR_UNSUPPORTED;
    AttnQ8Args a{};
    a.q = q; a.k_codes = (const uint8_t*)k_codes; a.v_codes = (const uint8_t*)v_codes; a.k_scales = k_scales;
    a.v_scales = v_scales; a.cu_seqlens = cu_seqlens; a.seq_end = seq_end; a.page_table = page_table;
    a.table_stride = table_stride; a.ring = ring; a.n_pages = n_pages; a.out = out; a.partial = partial;
    a.n_tokens = n_tokens; a.n_heads = n_heads; a.n_kv = n_kv; a.hd = hd; a.window = window; a.chunk = chunk;
    a.n_splits = n_splits; a.scale = scale; a.status = status;
    const int G = n_heads / n_kv, br = aq_block_rows(max_row_tokens, G, hd, dtype);
    const long long groups = ((long long)max_row_tokens * G + br - 1) / br;
    if (groups * n_kv > 65535) return MF_ERR_UNSUPPORTED;
    a.q_groups = (int)groups;
    const dim3 grid(n_splits, (unsigned)(groups * n_kv), n_rows);
    int e;
    if (aq_on_tensor_cores(hd, dtype)) {
        if (hd == 128)
            e = br == 16 ? (fmt == MF_Q8_E4M3 ? launch_mma<128, MF_Q8_E4M3, 1, 4, 3>(a, grid, stream)
                                              : launch_mma<128, MF_Q8_INT8, 1, 4, 3>(a, grid, stream))
                         : (fmt == MF_Q8_E4M3 ? launch_mma<128, MF_Q8_E4M3, 2, 4, 2>(a, grid, stream)
                                              : launch_mma<128, MF_Q8_INT8, 2, 4, 2>(a, grid, stream));
        else
            e = br == 16 ? (fmt == MF_Q8_E4M3 ? launch_mma<64, MF_Q8_E4M3, 1, 6, 4>(a, grid, stream)
                                              : launch_mma<64, MF_Q8_INT8, 1, 6, 4>(a, grid, stream))
                         : (fmt == MF_Q8_E4M3 ? launch_mma<64, MF_Q8_E4M3, 2, 6, 3>(a, grid, stream)
                                              : launch_mma<64, MF_Q8_INT8, 2, 6, 3>(a, grid, stream));
    } else if (dtype == MF_DTYPE_F32) {
        e = fmt == MF_Q8_E4M3 ? launch_generic<float, MF_Q8_E4M3>(a, grid, stream)
                              : launch_generic<float, MF_Q8_INT8>(a, grid, stream);
    } else {
        e = fmt == MF_Q8_E4M3 ? launch_generic<__nv_bfloat16, MF_Q8_E4M3>(a, grid, stream)
                              : launch_generic<__nv_bfloat16, MF_Q8_INT8>(a, grid, stream);
    }
    if (e || n_splits == 1) return e;
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
