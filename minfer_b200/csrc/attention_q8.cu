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
// one matrix product, r = token * group + head.  (Portions of many tokens have a kernel on tcgen05,
// attention_q8_tc.cu.)
#include "q8.cuh"

#include <cooperative_groups.h>
#include <type_traits>

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
    float* partial;                // scratch, see the kernels
    int n_tokens, n_rows, n_heads, n_kv, hd, window;
    int max_end;                   // positions that the page table has room for
    int n_splits;                  // parts that a row's pages are shared out to
    int q_groups;                  // blocks along the longest row's matrix rows
    int block_rows;                // matrix rows a block takes
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
// A warp owns KT * 16 neighbouring keys of every KT pages of its block's split (four warps) and streams
// them through a ring of its own in shared memory, filled by cp.async: no barrier between warps until
// the end, where the four results are joined.  An 8-bit code is an exact half, so both products run on
// halves: the block's queries are brought below 2^15 by one power of two first (a half has more mantissa
// than a bfloat16, and 2^-28 of their largest element is still exact), the power goes into the
// float32 factor of the scores.
//
// Values' scales differ from key to key, and a half holds 2^-14..2^16: so what a row's exponentials are
// taken against is not its largest score but the largest weight so far, m = max_j (s_j + log2 vs_j), and what
// is rounded to halves is 2^(s_j - m) vs_j (off by 2^-11, where a bfloat16 probability is off by 2^-8); the sum
// of 2^(s_j - m) is float32.  m is moved up (and outputs rescaled) only when a weight passes it by more than
// 2^10: nothing is near overflow until then, and the usual step needs one vote and no exchange between
// lanes.
//
// Bound by bytes where rows are few and caches long: 64 sequences of 2,047 to 8,100 positions, one token each, 28
// heads, 4 of keys, 128: 65 us, 5.3 TB/s (0.81 of a copy), the first pages' latency and the join included.  Where rows are many, a step of 16 keys takes a warp about 1,650 clocks
// at 24 rows (16 sequences with 4 drafts each over 1,501 to 3,001 positions: 30.8 us): its loads, conversions, products and
// exponentials follow one another, and two or three warps a scheduler do not hide them all.  Short calls are
// latency (8 sequences of 1,801 to 2,047 positions: 10.3 us).
//
// Layouts: row r of a score tile is key 4 (r' >> 1) + 2 (r >> 3) + (r & 1), r' = r & 7, of the step's 16, so that
// the keys a thread multiplies values of are the four from 4 t on.  Both operands of a score see the same
// order of dimensions (a thread takes 16 neighbouring codes of a key: one load feeds four k-steps); rows g and
// g + 8 of output tile j are dimensions (HD / 8) g + 2 j and + 1, so a thread ends up with HD / 8 neighbouring ones.
// ------------------------------------------------------------------------------------------
#define AQ_WARPS 4
#define AQ_KEYS 16
#define AQ_WEIGHT_ROOM 1024.0f    // a weight beyond it moves the reference
#define AQ_SCORE_ROOM 100.0f      // so does 2^100 without a value's scale (which may be zero)

template <int HD> struct AqTile {                          // 16 keys: K, V, scales
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
#define AQ_WHOLE 0
#define AQ_SPLIT 1
#define AQ_SHARED 2
#define AQ_LEAST_PAGES 2          // that a block of AQ_SHARED takes

// What a row of the batch asks for: its tokens and pages, and how many pages all its items have.
struct AqRow {
    int tok0, count, end, base0, pages, items;
};
// A row's tokens and its end, brought inside what there is (numbers that the device gave may be anything; an end
// behind the page table is reported, and tokens in front of position 0 see nothing).
__device__ __forceinline__ void aq_bounds(const AttnQ8Args& a, int b, int* tok0, int* count, int* end) {
    const int from = a.cu_seqlens[b], to = a.cu_seqlens[b + 1], e = a.seq_end[b];
    *tok0 = from;
    *count = from >= 0 && from <= to && to <= a.n_tokens ? to - from : 0;
    *end = min(max(e, 0), a.max_end);
    if (e > a.max_end && *count > 0 && threadIdx.x == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
}
__device__ __forceinline__ AqRow aq_row(const AttnQ8Args& a, int b, int rows_a_block) {
    AqRow r;
    aq_bounds(a, b, &r.tok0, &r.count, &r.end);
    const int first = r.end - r.count;
    r.base0 = (a.window > 0 ? max(0, first - a.window + 1) : 0) & ~(MF_PAGE - 1);
    r.items = a.n_kv * min(a.q_groups, (r.count * (a.n_heads / a.n_kv) + rows_a_block - 1) / rows_a_block);
    // (a row that sees nothing still has zeros to write: one page, which no key of it is in)
    r.pages = r.count > 0 ? max(1, (r.end - r.base0 + MF_PAGE - 1) / MF_PAGE) : 0;
    return r;
}
// AQ_SHARED: block c of n takes pages [c s, (c + 1) s) of all U, s = ceil(U / n).
__device__ __forceinline__ int aq_share(int units, int blocks) {
    return max(AQ_LEAST_PAGES, (units + blocks - 1) / blocks);
}
// Its scratch: for every block where its first page lies and s, then two results a block (of an item begun by
// another block, and of one begun here that another ends): [rows][HD] outputs, then maxima and sums.
struct __align__(16) AqFirst {
    int row, item, page0, share;               // share 0: the block has no pages
};
__host__ __device__ constexpr size_t aq_slot_floats(int rows, int hd) { return (size_t)rows * (hd + 2); }
__host__ __device__ constexpr size_t aq_table_floats(int blocks) { return (size_t)blocks * 4; }

__device__ __forceinline__ float over_keys_max(float v) {             // over the eight lanes of one t
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}

// NT: tiles of 8 matrix rows a block takes; KT: tiles of 16 keys a warp takes at a time.  An item is one
// (row of the batch, key/value head, 8 NT matrix rows).  How items are shared out:
//   AQ_WHOLE    a block an item
//   AQ_SPLIT    an item's pages are split among the blocks of a cluster, which join their results through
//               distributed shared memory: one launch, for calls whose blocks are all on the GPU at once
//   AQ_SHARED   the pages of all items, one behind the other, are dealt out evenly to as many blocks as the
//               GPU holds, wherever one item ends and the next begins; items that several blocks have
//               worked on are joined by attention_q8_join_kernel.  Rows of any lengths keep every SM busy
//               to the end.
template <int HD, int FMT, int NT, int KT, int MODE, int STAGES, int MINB>
__global__ void __launch_bounds__(AQ_WARPS * 32, MINB) attention_q8_mma_kernel(AttnQ8Args a) {
    using T = AqTile<HD>;
    namespace cg = cooperative_groups;
    constexpr int OT = HD / 16;                            // output tiles of 16 dimensions
    constexpr int OS = HD + 4;                             // floats a row of the joining buffer
    constexpr int ROWS = 8 * NT;
    extern __shared__ __align__(128) uint8_t aq_smem[];
    __shared__ float2 ml_s[AQ_WARPS][ROWS];
    __shared__ float f_s[AQ_WARPS][ROWS];
    __shared__ float2 row_s[ROWS];                         // the block's maximum and sum of each row
    pdl_launch_dependents();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int G = a.n_heads / a.n_kv;

    // ---- which pages of which items ----
    int b = blockIdx.z, item = MODE == AQ_WHOLE ? blockIdx.x : blockIdx.y, page0 = 0, page1 = 0;          // pages [page0, page1) of the item
    int todo = 0;                                                         // AQ_SHARED: pages left to this block
    AqFirst first_of;
    AqRow row;
    if constexpr (MODE == AQ_SHARED) {
        // the pages in front of every row and in all, then the row that the block's first page belongs to
        __shared__ int scan_s[AQ_WARPS], at_s[2];
        int units = 0, before = 0, share = 0, begin = 0;
        for (int b0 = 0; b0 < a.n_rows;) {
            int mine = 0;
            if (b0 + tid < a.n_rows) {
                const AqRow r = aq_row(a, b0 + tid, ROWS);
                mine = r.pages * r.items;
            }
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            __syncthreads();
            if (lane == 31) scan_s[warp] = upto;
            __syncthreads();
            int all = 0;
#pragma unroll
            for (int w = 0; w < AQ_WARPS; ++w) {
                if (w < warp) upto += scan_s[w];
                all += scan_s[w];
            }
            const bool known = share > 0;                                 // (the second time through)
            if (!known) units += all;
            const bool done = !known && b0 + AQ_WARPS * 32 >= a.n_rows;
            if (done) {
                share = aq_share(units, gridDim.x);
                begin = blockIdx.x * share;
                todo = min(share, units - begin);
            }
            if (known || a.n_rows <= AQ_WARPS * 32) {
                const int from = before + upto - mine;
                if (mine > 0 && from <= begin && begin < from + mine) { at_s[0] = b0 + tid; at_s[1] = from; }
                before += all;
            }
            b0 += AQ_WARPS * 32;
            if (done && a.n_rows > AQ_WARPS * 32 && todo > 0) b0 = 0;     // once more, with the block's page known
        }
        __syncthreads();
        AqFirst* firsts = (AqFirst*)a.partial;
        if (todo <= 0) {
            // (what a kernel before this one may still read of its own scratch is not touched before it has ended)
            pdl_wait();
            if (tid == 0) firsts[blockIdx.x].share = 0;
            return;
        }
        b = at_s[0];
        row = aq_row(a, b, ROWS);
        item = (begin - at_s[1]) / row.pages;
        page0 = begin - at_s[1] - item * row.pages;
        first_of.row = b; first_of.item = item; first_of.page0 = page0; first_of.share = share;
    } else {
        row = aq_row(a, b, ROWS);
        // (uniform over a cluster)
        if (item >= row.items) { pdl_wait(); return; }
        const int chunk = MODE == AQ_SPLIT ? (row.pages + a.n_splits - 1) / a.n_splits : row.pages;
        page0 = MODE == AQ_SPLIT ? min(row.pages, (int)blockIdx.x * chunk) : 0;
        page1 = min(row.pages, page0 + chunk);
    }
    bool waited = false;

    for (;;) {
    if constexpr (MODE == AQ_SHARED) page1 = min(row.pages, page0 + todo);
    const int tok0 = row.tok0, count = row.count, end = row.end;
    const int hk = item % a.n_kv, qg = item / a.n_kv;
    const int r0 = qg * ROWS, rows = min(ROWS, count * G - r0);           // the block's matrix rows
    // what the block's queries see together: [lo, hi); and every one of them: [lo_in, hi_in)
    const int first = end - count + r0 / G, last = end - count + (r0 + rows - 1) / G;
    const int lo_all = a.window > 0 ? max(0, first - a.window + 1) : 0;
    const int lo_in = a.window > 0 ? max(0, last - a.window + 1) : 0, hi_in = first + 1;
    const int base = row.base0 + page0 * MF_PAGE;
    const int lo = max(lo_all, base), hi = min(last + 1, row.base0 + page1 * MF_PAGE);
    const int n_it = hi > lo ? (hi - base + KT * MF_PAGE - 1) / (KT * MF_PAGE) : 0;
    const int* table = a.page_table + (size_t)b * a.table_stride;

    // ---- the ring ----
    constexpr int STAGE = KT * T::STAGE;
    const uint32_t ring0 = (uint32_t)__cvta_generic_to_shared(aq_smem) + warp * STAGES * STAGE;
    const int key0 = base + warp * KT * AQ_KEYS;           // the warp's first key of iteration 0
    const int in_page = key0 & (MF_PAGE - 1);
    int ids = -1;                              // lane i: the page of iteration (it & ~31) + i
    unsigned there = 0, there_next = 0;        // bit i: so many iterations on, that page is one
    auto look_up = [&](int it) {               // the next 32 page numbers
        const int p = key0 + (it + lane) * KT * MF_PAGE;
        const int index = (a.ring > 0 ? p % a.ring : p) >> 6;
        const bool seen = p < hi && p + KT * AQ_KEYS > lo;
        ids = seen && index < a.table_stride ? table[index] : -1;
        const bool page = ids >= 0 && ids < a.n_pages;
        // a page that is not there: its keys are seen by nobody, and the caller is told
        if (seen && !page) atomicOr(a.status, MF_STATUS_BAD_POSITION);
        there_next = __ballot_sync(0xffffffffu, page);
    };
    look_up(0);
    there = there_next;
    // what a lane copies, from the pages' beginnings on
    const size_t vectors = (size_t)hk * MF_PAGE + in_page;
    const uint8_t* const k_from = a.k_codes + vectors * HD + lane * 16;
    const uint8_t* const v_from = a.v_codes + vectors * HD + lane * 16;
    const float* const s_from = (lane < 4 ? a.k_scales : a.v_scales - 16) + vectors + lane * 4;
    const size_t page_vectors = (size_t)a.n_kv * MF_PAGE;
    const uint32_t k_lane = T::k_at(lane / T::CPR, lane % T::CPR), v_lane = T::CODES + T::v_at(lane / T::CPR, lane % T::CPR);
    uint32_t fetch_to = ring0;
    if (!waited) {
        pdl_wait();
        if (MODE == AQ_SHARED && tid == 0) ((AqFirst*)a.partial)[blockIdx.x] = first_of;
    }
    waited = true;
    auto fetch = [&](int it) {
        if ((it & 31) == 0 && it > 0) look_up(it);
        if (it < n_it && ((there_next >> (it & 31)) & 1u)) {
            const size_t at = (size_t)__shfl_sync(0xffffffffu, ids, it & 31) * page_vectors;
            const uint8_t* kp = k_from + at * HD;
            const uint8_t* vp = v_from + at * HD;
#pragma unroll
            for (int k = 0; k < KT; ++k) {
#pragma unroll
                for (int i = 0; i < AQ_KEYS * T::CPR / 32; ++i) {
                    // row lane / CPR + (32 / CPR) i: a multiple of 2 further, so that K's permutation is the
                    // lane's; V's changes by the rows' quads (stages are multiples of 128 bytes)
                    constexpr int V_STEP = HD == 128 ? 32 : 64;
                    cp16(fetch_to + k * T::STAGE + k_lane + i * 512, kp + (k * AQ_KEYS * HD + i * 512));
                    cp16(((fetch_to + k * T::STAGE + v_lane) ^ (i * V_STEP)) + i * 512, vp + (k * AQ_KEYS * HD + i * 512));
                }
                if (lane < 8) cp16(fetch_to + k * T::STAGE + 2 * T::CODES + lane * 16, s_from + at + k * AQ_KEYS);
            }
        }
        fetch_to = fetch_to == ring0 + (STAGES - 1) * STAGE ? ring0 : fetch_to + STAGE;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i);

    // ---- queries: a thread loads a part of row g of each tile; it works on the scores of rows 2 t, 2 t + 1 ----
    uint32_t qb[NT][HD / 16][2];
    float neg[NT][2];                          // minus the reference: infinity before the first key, NaN for a
                                               // row that holds what is not finite
    float c_q;                                 // scale log2(e) / the queries' power of two
    {
        uint4 w[NT][HD / 64][2];
        unsigned top = 0;
        bool bad[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 8 + g;
            if (r < rows) {
                const int token = (r0 + r) / G, head = hk * G + (r0 + r) - token * G;
                const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + ((size_t)(tok0 + token) * a.n_heads + head) * HD;
#pragma unroll
                for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                    for (int i = 0; i < 2; ++i) w[n][c][i] = *reinterpret_cast<const uint4*>(q + 64 * c + 16 * t + 8 * i);
            } else {
#pragma unroll
                for (int c = 0; c < HD / 64; ++c) w[n][c][0] = w[n][c][1] = make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            unsigned mine = 0;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t x[4] = {w[n][c][i].x, w[n][c][i].y, w[n][c][i].z, w[n][c][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) mine = max(mine, max(x[j] & 0x7fffu, (x[j] >> 16) & 0x7fffu));
                }
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 2));
            bad[n] = mine >= 0x7f80u;
            if (!bad[n]) top = max(top, mine);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        // the power of two: 2^(14 - exponent), from the exponent field (0: zeros or numbers below the normal
        // range, which 2^100 brings up and which count as zero below 2^-124)
        const int field = (int)(top >> 7);
        const int power = field == 0 ? 100 : min(141 - field, 100);
        const float up = __int_as_float((power + 127) << 23), down = __int_as_float((127 - power) << 23);
        c_q = a.scale * 1.4426950408889634f * down;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                neg[n][i] = __shfl_sync(0xffffffffu, bad[n] ? __int_as_float(0x7fc00000) : INFINITY, (2 * t + i) * 4);
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t x[4] = {w[n][c][i].x, w[n][c][i].y, w[n][c][i].z, w[n][c][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float f0 = bad[n] ? 0.0f : __uint_as_float(x[j] << 16) * up;
                        const float f1 = bad[n] ? 0.0f : __uint_as_float(x[j] & 0xffff0000u) * up;
                        // elements 8 i + 2 j, + 1 of the thread's 16: k-step 2 i + j / 2, first or second pair
                        qb[n][4 * c + 2 * i + (j >> 1)][j & 1] = pack_half2(f0, f1);
                    }
                }
        }
    }

    float l_q[NT][2], o[NT][OT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        l_q[n][0] = l_q[n][1] = 0.0f;
#pragma unroll
        for (int j = 0; j < OT; ++j) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.0f;
    }

    const int key_a = 4 * (g >> 1) + (g & 1);              // the thread's keys: this one and the one 2 behind
    const uint32_t ka_at = T::k_at(key_a, t), kb_at = T::k_at(key_a + 2, t);
    const uint32_t v_at0 = T::CODES + (HD == 128 ? T::v_at(4 * t, g) : T::v_at(4 * t, g >> 1) + 8 * (g & 1));
    const uint32_t s_at = 2 * T::CODES + key_a * 4;
    uint32_t stage = ring0;

    // 16 KT keys from position k0 on.  EDGE: some of them are not seen by some of the rows.
    auto step = [&](auto edge_tag, int k0) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        float sc[KT][NT][4];
#pragma unroll
        for (int k = 0; k < KT; ++k) {
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[k][n][0] = sc[k][n][1] = sc[k][n][2] = sc[k][n][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                // (the second 64 dimensions lie in the other half of 128 bytes)
                const uint4 ka = lds128((stage + k * T::STAGE + ka_at) ^ (c * 64)), kb = lds128((stage + k * T::STAGE + kb_at) ^ (c * 64));
                const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t x = q8_prepare<FMT>(wa[j]), y = q8_prepare<FMT>(wb[j]);
                    const uint32_t af[4] = {q8_halves<FMT, false>(x), q8_halves<FMT, false>(y), q8_halves<FMT, true>(x),
                                            q8_halves<FMT, true>(y)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(sc[k][n], af, qb[n][4 * c + j][0], qb[n][4 * c + j][1]);
                }
            }
        }
        float ks[KT][2], vs[KT][2];
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                ks[k][u] = lds32(stage + k * T::STAGE + s_at + 8 * u) * c_q;
                vs[k][u] = lds32(stage + k * T::STAGE + s_at + 64 + 8 * u);
            }
        // bit 2 u + i of gone[k][n]: row i of tile n does not see key u of tile k
        unsigned gone[KT][NT];
        if constexpr (EDGE) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                int to[2], from[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = n * 8 + 2 * t + i, pos = r < rows ? end - count + (r0 + r) / G : -1;
                    to[i] = min(pos + 1, hi);
                    from[i] = a.window > 0 ? max(lo, pos - a.window + 1) : lo;
                }
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    gone[k][n] = 0;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int at = k0 + k * AQ_KEYS + key_a + 2 * u;
                            if (at >= to[i] || at < from[i]) gone[k][n] |= 1u << (2 * u + i);
                        }
                }
            }
        }
        float x[KT][NT][4], w[KT][NT][4];
        float most = AQ_NEG, heaviest = 0.0f;
        // AGAIN: with references of this step's scores.  A fused difference is off by what the reference was rounded by,
        // which beyond 2^30 is more than a float's range of powers: then scores are rounded first, as references were
        auto weigh = [&](auto again_tag) {
#pragma unroll
            for (int k = 0; k < KT; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {          // 2 key + row
                        x[k][n][e] = decltype(again_tag)::value ? __fadd_rn(__fmul_rn(sc[k][n][e], ks[k][e >> 1]), neg[n][e & 1])
                                                                : fmaf(sc[k][n][e], ks[k][e >> 1], neg[n][e & 1]);
                        // (a key or value that is not seen may have any scale: NaN must not get in)
                        if (EDGE && ((gone[k][n] >> e) & 1u)) x[k][n][e] = AQ_NEG;
                        w[k][n][e] = ex2(x[k][n][e]) * vs[k][e >> 1];
                        if (EDGE && ((gone[k][n] >> e) & 1u)) w[k][n][e] = 0.0f;
                        most = fmaxf(most, x[k][n][e]);
                        heaviest = fmaxf(heaviest, w[k][n][e]);
                    }
        };
        weigh(std::false_type{});
        if (__any_sync(0xffffffffu, most > AQ_SCORE_ROOM || heaviest > AQ_WEIGHT_ROOM)) {
            // the references up to what is known now: the largest score first, then the largest weight
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float top = AQ_NEG, big = 0.0f;
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (!EDGE || !((gone[k][n] >> (2 * u + i)) & 1u)) top = fmaxf(top, __fmul_rn(sc[k][n][2 * u + i], ks[k][u]));
                    const float before = -neg[n][i];
                    top = over_keys_max(top);
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                            if (!EDGE || !((gone[k][n] >> (2 * u + i)) & 1u))
                                big = fmaxf(big, ex2(__fadd_rn(__fmul_rn(sc[k][n][2 * u + i], ks[k][u]), -top)) * vs[k][u]);
                    big = fmaxf(over_keys_max(big), 8.1e-28f);         // (2^-90: values of zeros)
                    // (a row that has seen nothing yet keeps its infinity, one that is NaN its NaN)
                    const float m = fmaxf(before, top + __log2f(big));
                    const float f = before == AQ_NEG ? 0.0f : ex2(before - m);
                    if (top > AQ_NEG && before == before) neg[n][i] = -m;
                    l_q[n][i] *= f;
#pragma unroll
                    for (int j = 0; j < OT; ++j) { o[n][j][i] *= f; o[n][j][2 + i] *= f; }
                }
            weigh(std::true_type{});
        }
        uint32_t pb[KT][NT][2];
#pragma unroll
        for (int k = 0; k < KT; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) l_q[n][i] += ex2(x[k][n][i]) + ex2(x[k][n][2 + i]);
                pb[k][n][0] = transposed(pack_half2(w[k][n][0], w[k][n][1]));
                pb[k][n][1] = transposed(pack_half2(w[k][n][2], w[k][n][3]));
            }
        // ---- values: pairs of keys of one dimension, HD / 8 dimensions of the keys 4 t .. 4 t + 3 ----
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            uint32_t vw[4][HD / 32];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t v0 = stage + k * T::STAGE + v_at0;
                const uint32_t at = HD == 128 ? v0 + i * 128 : (v0 ^ ((i & 1) * 64)) + (i >> 1) * 128;
                if constexpr (HD == 128) {
                    const uint4 v = lds128(at);
                    vw[i][0] = v.x; vw[i][1] = v.y; vw[i][2] = v.z; vw[i][3] = v.w;
                } else {
                    const uint2 v = lds64(at);
                    vw[i][0] = v.x; vw[i][1] = v.y;
                }
                // codes of places that no query of the block sees are anybody's
                if (EDGE && (k0 + k * AQ_KEYS + 4 * t + i < lo || k0 + k * AQ_KEYS + 4 * t + i >= hi))
#pragma unroll
                    for (int h = 0; h < HD / 32; ++h) vw[i][h] = 0u;
            }
#pragma unroll
            for (int h = 0; h < HD / 32; ++h)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t y = q8_prepare<FMT>(__byte_perm(vw[0][h], vw[1][h], u ? 0x7362 : 0x5140));
                    const uint32_t z = q8_prepare<FMT>(__byte_perm(vw[2][h], vw[3][h], u ? 0x7362 : 0x5140));
                    const uint32_t af[4] = {q8_halves<FMT, false>(y), q8_halves<FMT, true>(y), q8_halves<FMT, false>(z),
                                            q8_halves<FMT, true>(z)};
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[n][2 * h + u], af, pb[k][n][0], pb[k][n][1]);
                }
        }
    };

    const int lo_edge = max(lo_in, lo), hi_edge = min(hi_in, hi) - KT * AQ_KEYS;
    for (int it = 0; it < n_it; ++it) {
        if ((it & 31) == 0 && it > 0) there = there_next;
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
        if ((there >> (it & 31)) & 1u) {
            const int k0 = key0 + it * KT * MF_PAGE;
            if (k0 < lo_edge || k0 > hi_edge) step(std::true_type{}, k0);
            else step(std::false_type{}, k0);
        }
        __syncwarp();                          // the stage the next fetch fills was read an iteration ago
        fetch(it + STAGES - 1);
        stage = stage == ring0 + (STAGES - 1) * STAGE ? ring0 : stage + STAGE;
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
            // (a row that holds what is not finite: its reference is NaN, its sum too)
            const bool bad = neg[n][i] != neg[n][i];
            if (g == 0) ml_s[warp][n * 8 + 2 * t + i] = make_float2(bad ? AQ_NEG : -neg[n][i], bad ? neg[n][i] : l);
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
        for (int w = 0; w < AQ_WARPS; ++w) m = fmaxf(m, ml_s[w][tid].x);
        const float m_use = m == AQ_NEG ? 0.0f : m;
#pragma unroll
        for (int w = 0; w < AQ_WARPS; ++w) {
            const float f = exp2f(ml_s[w][tid].x - m_use);
            f_s[w][tid] = f;
            l += ml_s[w][tid].y * f;
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
    if constexpr (MODE == AQ_SPLIT) {
        cg::cluster_group cluster = cg::this_cluster();
        const int n = a.n_splits, rank = blockIdx.x;
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
        return;
    } else {
        if (MODE == AQ_SHARED && (page0 > 0 || page1 < row.pages)) {
            // a part of the item: the first result if another block began it, else the second
            float* slot = a.partial + aq_table_floats(gridDim.x) + (2 * (size_t)blockIdx.x + (page0 > 0 ? 0 : 1)) * aq_slot_floats(ROWS, HD);
            for (int i = tid; i < units; i += AQ_WARPS * 32) {
                const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
                *reinterpret_cast<float4*>(slot + (size_t)r * HD + d) = joined(r, d);
            }
            for (int r = tid; r < rows; r += AQ_WARPS * 32)
                *reinterpret_cast<float2*>(slot + (size_t)ROWS * HD + 2 * r) = row_s[r];
        } else {
            for (int i = tid; i < units; i += AQ_WARPS * 32) {
                const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
                const float l = row_s[r].y;
                write_out(r, d, joined(r, d), l == 0.0f ? 0.0f : 1.0f / l);
            }
        }
        if constexpr (MODE != AQ_SHARED) return;
        todo -= page1 - page0;
        if (todo <= 0) return;
        // on to the next item
        page0 = 0;
        if (++item == row.items) {
            item = 0;
            do row = aq_row(a, ++b, ROWS); while (row.pages == 0);
        }
        __syncthreads();                       // everybody is done with the joined results
    }
    }
}

// Items that several blocks of AQ_SHARED have worked on: their results joined in the blocks' order.  Block c of a
// row r of the grid joins matrix row r of the item that block c of the attention kernel began in, if it was the
// second to work on it: its warps share the results out, a lane takes four dimensions.
#define AQ_JOIN_WARPS 4
template <int HD, int ROWS>
__global__ void __launch_bounds__(AQ_JOIN_WARPS * 32) attention_q8_join_kernel(AttnQ8Args a, int blocks) {
    pdl_launch_dependents();
    __shared__ float4 acc_s[AQ_JOIN_WARPS][HD / 4];
    __shared__ float2 ml_s[AQ_JOIN_WARPS];
    const int c = blockIdx.x + 1, r = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    const AqFirst at_c = ((const AqFirst*)a.partial)[c];
    if (at_c.share == 0 || at_c.page0 == 0 || at_c.page0 > at_c.share) return;
    const AqRow row = aq_row(a, at_c.row, ROWS);
    const int G = a.n_heads / a.n_kv, hk = at_c.item % a.n_kv, at = at_c.item / a.n_kv * ROWS + r;
    if (at >= row.count * G) return;
    const int c0 = c - 1, c1 = c + (row.pages - at_c.page0 - 1) / at_c.share;
    const float* slots = a.partial + aq_table_floats(blocks);
    auto slot = [&](int c) { return slots + (2 * (size_t)c + (c == c0 ? 1 : 0)) * aq_slot_floats(ROWS, HD); };
    const bool mine = lane < HD / 4;
    float m = AQ_NEG, l = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int first = c0 + warp; first <= c1; first += 4 * AQ_JOIN_WARPS) {
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = first + AQ_JOIN_WARPS * i;
            ml[i] = make_float2(AQ_NEG, 0.0f);
            x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (c <= c1) {
                ml[i] = *reinterpret_cast<const float2*>(slot(c) + ROWS * HD + 2 * r);
                if (mine) x[i] = *reinterpret_cast<const float4*>(slot(c) + (size_t)r * HD + 4 * lane);
            }
        }
        const float top = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
        const float m_use = top == AQ_NEG ? 0.0f : top, keep = exp2f(m - m_use);
        m = top;
        l *= keep;
        acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float f = exp2f(ml[i].x - m_use);
            l = fmaf(ml[i].y, f, l);
            acc.x = fmaf(x[i].x, f, acc.x); acc.y = fmaf(x[i].y, f, acc.y);
            acc.z = fmaf(x[i].z, f, acc.z); acc.w = fmaf(x[i].w, f, acc.w);
        }
    }
    if (mine) acc_s[warp][lane] = acc;
    if (lane == 0) ml_s[warp] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= HD / 4) return;
    float top = AQ_NEG, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < AQ_JOIN_WARPS; ++w) top = fmaxf(top, ml_s[w].x);
    const float m_use = top == AQ_NEG ? 0.0f : top;
    float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < AQ_JOIN_WARPS; ++w) {
        const float f = exp2f(ml_s[w].x - m_use);
        const float4 x = acc_s[w][threadIdx.x];
        sum = fmaf(ml_s[w].y, f, sum);
        out.x = fmaf(x.x, f, out.x); out.y = fmaf(x.y, f, out.y);
        out.z = fmaf(x.z, f, out.z); out.w = fmaf(x.w, f, out.w);
    }
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int token = at / G, head = hk * G + at - token * G;
    const __nv_bfloat162 x = __floats2bfloat162_rn(out.x * by, out.y * by);
    const __nv_bfloat162 y = __floats2bfloat162_rn(out.z * by, out.w * by);
    *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)(row.tok0 + token) * a.n_heads + head) * HD + 4 * threadIdx.x) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// ------------------------------------------------------------------------------------------
// Any head size that is a multiple of 16 up to 256, float32 or bfloat16 queries, in float32 on the
// FP32 pipe (the true 32-bit path).  A block takes up to eight matrix rows of one key/value head; 32
// keys at a time are turned into float32 codes in shared memory once for all of them, lanes are keys
// in the scores and dimensions in the sums; a warp's two rows share what it reads of keys and values.  Bound by
// the shared-memory reads of the products: 16 sequences over 4,000 positions, 28 heads, 4 of keys, 128: 146 us, 6
// TFLOP/s; few rows by latency (4 of 1 to 3 tokens over 60 to 611: 14.4 us, the join 3 of them).  ND: 32 dimensions a lane has one of, rounded up to 1, 2, 4 or 8.
// ------------------------------------------------------------------------------------------
#define AG_WARPS 4
#define AG_ROWS 8
#define AG_KEYS 32

// KEYS positions' codes, from vector `at` of the pages on, as float values or halves (exact both): keys in rows of
// hs elements, values of hd.  A thread's unit is 4 codes, so that stores meet every bank; places outside [n0, n1) are zeros (what they hold
// is anybody's).  `by_row`: 2^32 / (hd / 4), rounded up: a unit's row by one multiplication.
template <int FMT, int KEYS, typename E>
__device__ __forceinline__ void ag_load(const AttnQ8Args& a, long long at, int n0, int n1, E* k_s, int hs, E* v_s,
                                        unsigned by_row) {
    const int hd = a.hd, upr = hd >> 2, units = KEYS * upr;
#pragma unroll 1
    for (int u0 = threadIdx.x; u0 < 2 * units; u0 += 8 * 128) {
        uint32_t w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int u = u0 + j * 128, v = u >= units ? u - units : u, r = (int)__umulhi((unsigned)v, by_row);
            w[j] = 0;
            if (u < 2 * units && r >= n0 && r < n1)
                w[j] = reinterpret_cast<const uint32_t*>((u >= units ? a.v_codes : a.k_codes) + at * hd)[v];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int u = u0 + j * 128, v = u >= units ? u - units : u, r = (int)__umulhi((unsigned)v, by_row);
            if (u >= 2 * units) continue;
            E* to = u >= units ? v_s + 4 * v : k_s + r * hs + 4 * (v - r * upr);
            if constexpr (sizeof(E) == 4) {
                float f[4];
                q8_floats<FMT>(w[j], f);
                *reinterpret_cast<float4*>(to) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
                const uint32_t x = q8_prepare<FMT>(w[j]);
                *reinterpret_cast<uint2*>(to) = make_uint2(q8_halves<FMT, false>(x), q8_halves<FMT, true>(x));
            }
        }
    }
}
// ROWS matrix rows' queries times the scale, zeros behind the last; place_s: where a row lies among q and out.
template <typename T, int ROWS>
__device__ __forceinline__ void ag_queries(const AttnQ8Args& a, int tok0, int hk, int r0, int rows, size_t* place_s, float* q_s) {
    const int G = a.n_heads / a.n_kv, hd = a.hd;
    if (threadIdx.x < ROWS) {
        const int r = r0 + threadIdx.x, token = r / G;
        place_s[threadIdx.x] = (size_t)(tok0 + token) * a.n_heads + hk * G + r - token * G;
    }
    __syncthreads();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int j = 0; j < ROWS / 4; ++j) {
        const int r = warp + 4 * j;
        const T* from = (const T*)a.q + place_s[r] * hd;
        for (int d = lane; d < hd; d += 32) q_s[r * hd + d] = r < rows ? to_f32(from[d]) * a.scale : 0.0f;
    }
}

template <typename T, int FMT, int ND>
__global__ void __launch_bounds__(AG_WARPS * 32) attention_q8_generic_kernel(AttnQ8Args a, unsigned by_row) {
    extern __shared__ __align__(16) uint8_t ag_smem[];
    pdl_launch_dependents();
    __shared__ size_t place_s[AG_ROWS];
    const int hd = a.hd, hs = hd + 4;                      // rows of an odd number of 16 bytes: lanes meet every bank
    float* k_s = (float*)ag_smem;                          // [AG_KEYS][hs]
    float* v_s = k_s + AG_KEYS * hs;                       // [AG_KEYS][hd]
    float* q_s = v_s + AG_KEYS * hd;                       // [AG_ROWS][hd]
    float* ks_s = q_s + AG_ROWS * hd;                      // [AG_KEYS] each
    float* vs_s = ks_s + AG_KEYS;
    float* p_s = vs_s + AG_KEYS;                           // [AG_ROWS][AG_KEYS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = blockIdx.y, hk = blockIdx.x / a.q_groups, qg = blockIdx.x - hk * a.q_groups, b = blockIdx.z;
    const int G = a.n_heads / a.n_kv;
    int tok0, count, end;
    aq_bounds(a, b, &tok0, &count, &end);
    const int r0 = qg * AG_ROWS, rows = min(AG_ROWS, count * G - r0);
    if (rows <= 0) { pdl_wait(); return; }
    const int first = end - count + r0 / G, last = end - count + (r0 + rows - 1) / G;
    const int lo_all = a.window > 0 ? max(0, first - a.window + 1) : 0;
    const int base0 = lo_all & ~(MF_PAGE - 1), pages = max(0, (last - base0 + MF_PAGE) / MF_PAGE);
    const int chunk = (pages + a.n_splits - 1) / a.n_splits * MF_PAGE;
    const int base = base0 + split * chunk;
    const int lo = max(lo_all, base), hi = min(last + 1, base + chunk);
    const int* table = a.page_table + (size_t)b * a.table_stride;
    pdl_wait();
    ag_queries<T, AG_ROWS>(a, tok0, hk, r0, rows, place_s, q_s);
    constexpr int RW = AG_ROWS / AG_WARPS;                 // rows a warp
    static_assert(RW == 2, "a warp's weights are read as pairs");
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
        ag_load<FMT, AG_KEYS>(a, at, lo - j0, hi - j0, k_s, hs, v_s, by_row);
        if (tid < AG_KEYS) ks_s[tid] = a.k_scales[at + tid];
        else if (tid < 2 * AG_KEYS) vs_s[tid - AG_KEYS] = a.v_scales[at + tid - AG_KEYS];
        __syncthreads();
        const int j = j0 + lane;
        bool seen[RW], any = false;
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            seen[i] = j >= max(lo_w[i], lo) && j < min(hi_w[i], hi);
            any |= seen[i];
        }
        if (!__any_sync(0xffffffffu, any)) continue;
        const float* kr = k_s + lane * hs;
        const float* qr = q_s + warp * RW * hd;
        float dot[RW][4];
#pragma unroll
        for (int i = 0; i < RW; ++i) dot[i][0] = dot[i][1] = dot[i][2] = dot[i][3] = 0.0f;
#pragma unroll 4
        for (int d = 0; d < hd; d += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
            for (int i = 0; i < RW; ++i) {
                const float4 q4 = *reinterpret_cast<const float4*>(qr + i * hd + d);
                dot[i][0] = fmaf(q4.x, k4.x, dot[i][0]); dot[i][1] = fmaf(q4.y, k4.y, dot[i][1]);
                dot[i][2] = fmaf(q4.z, k4.z, dot[i][2]); dot[i][3] = fmaf(q4.w, k4.w, dot[i][3]);
            }
        }
#pragma unroll
        for (int i = 0; i < RW; ++i) {
            const float s = seen[i] ? ((dot[i][0] + dot[i][1]) + (dot[i][2] + dot[i][3])) * ks_s[lane] : AQ_NEG;
            const float top = fmaxf(m_r[i], warp_max(s));
            const float m_use = top == AQ_NEG ? 0.0f : top;
            const float f = expf(m_r[i] - m_use), p = expf(s - m_use);
            l_r[i] = l_r[i] * f + warp_sum(p);
            m_r[i] = top;
            p_s[(warp * AG_KEYS + lane) * RW + i] = seen[i] ? p * vs_s[lane] : 0.0f;
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[i][d] *= f;
        }
        __syncwarp();
#pragma unroll 8
        for (int jj = 0; jj < AG_KEYS; ++jj) {
            const float2 w = *reinterpret_cast<const float2*>(p_s + (warp * AG_KEYS + jj) * RW);
#pragma unroll
            for (int d = 0; d < ND; ++d)
                if (32 * d + 32 <= hd || lane + 32 * d < hd) {
                    const float v = v_s[jj * hd + lane + 32 * d];
                    acc[0][d] = fmaf(w.x, v, acc[0][d]);
                    acc[1][d] = fmaf(w.y, v, acc[1][d]);
                }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < RW; ++i) {
        const int r = warp * RW + i;
        if (r >= rows) continue;
        const size_t th = place_s[r];
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
// The same for many matrix rows: a block takes 32 rows and 64 keys at a time.  Scores and outputs are formed in
// tiles of registers, since shared memory gives a warp 128 bytes a clock however few addresses it asks for: a thread
// has 4 rows by 4 keys and 4 rows by hd / 16 dimensions; sixteen lanes of a warp share four rows, so weights pass
// between them without a barrier of the block.  Codes lie in shared memory as halves (exact), which lets three
// blocks share an SM (as floats two: 16 sequences of 4 tokens behind 2,000, 40 heads, 8 of keys, 128: 246 us, 378
// with floats).  12 TFLOP/s of 72: loads are waited for in front of each page, and three blocks do not hide that.
// NJ: 64 dimensions, rounded up.
// ------------------------------------------------------------------------------------------
#define AM_ROWS 32
#define AM_KEYS 64
#define AM_LEAST 12            // rows beyond which a block takes 32
__device__ __forceinline__ float4 am_floats(const __half* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), y = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(x.x, x.y, y.x, y.y);
}
template <typename T, int FMT, int NJ>
__global__ void __launch_bounds__(128) attention_q8_rows_kernel(AttnQ8Args a, unsigned by_row) {
    extern __shared__ __align__(16) uint8_t ag_smem[];
    pdl_launch_dependents();
    const int hd = a.hd, hs = hd + 4;                      // rows of an odd number of 8 bytes: lanes meet every bank
    __half* k_s = (__half*)ag_smem;                        // [AM_KEYS][hs]
    __half* v_s = k_s + AM_KEYS * hs;                      // [AM_KEYS][hd]
    float* q_s = (float*)(v_s + AM_KEYS * hd);             // [AM_ROWS][hd]
    float* ks_s = q_s + AM_ROWS * hd;                      // [AM_KEYS] each
    float* vs_s = ks_s + AM_KEYS;
    float4* p_s = (float4*)(vs_s + AM_KEYS);               // [8][AM_KEYS]: the weights of four rows
    __shared__ size_t place_s[AM_ROWS];
    const int tid = threadIdx.x, rg = tid >> 4, kg = tid & 15;
    const int split = blockIdx.y, hk = blockIdx.x / a.q_groups, qg = blockIdx.x - hk * a.q_groups, b = blockIdx.z;
    const int G = a.n_heads / a.n_kv;
    int tok0, count, end;
    aq_bounds(a, b, &tok0, &count, &end);
    const int r0 = qg * AM_ROWS, rows = min(AM_ROWS, count * G - r0);
    if (rows <= 0) { pdl_wait(); return; }
    const int first = end - count + r0 / G, last = end - count + (r0 + rows - 1) / G;
    const int lo_all = a.window > 0 ? max(0, first - a.window + 1) : 0;
    const int base0 = lo_all & ~(MF_PAGE - 1), pages = max(0, (last - base0 + MF_PAGE) / MF_PAGE);
    const int chunk = (pages + a.n_splits - 1) / a.n_splits * MF_PAGE;
    const int base = base0 + split * chunk;
    const int lo = max(lo_all, base), hi = min(last + 1, base + chunk);
    const int* table = a.page_table + (size_t)b * a.table_stride;
    pdl_wait();
    ag_queries<T, AM_ROWS>(a, tok0, hk, r0, rows, place_s, q_s);
    float m_r[4], l_r[4], acc[4][4 * NJ];
    int lo_w[4], hi_w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m_r[i] = AQ_NEG; l_r[i] = 0.0f;
        const int r = rg * 4 + i;
        hi_w[i] = r < rows ? end - count + (r0 + r) / G + 1 : 0;
        lo_w[i] = r < rows && a.window > 0 ? max(0, hi_w[i] - a.window) : 0;
#pragma unroll
        for (int d = 0; d < 4 * NJ; ++d) acc[i][d] = 0.0f;
    }
    for (int j0 = lo & ~(AM_KEYS - 1); j0 < hi; j0 += AM_KEYS) {             // a page a step
        const int index = (a.ring > 0 ? j0 % a.ring : j0) >> 6;
        const int page = index < a.table_stride ? table[index] : -1;
        if (page < 0 || page >= a.n_pages) {                                 // (uniform over the block)
            if (tid == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
            continue;
        }
        const long long at = ((long long)page * a.n_kv + hk) * MF_PAGE;
        __syncthreads();                                   // the step before is done with the buffers
        ag_load<FMT, AM_KEYS>(a, at, lo - j0, hi - j0, k_s, hs, v_s, by_row);
        if (tid < AM_KEYS) ks_s[tid] = a.k_scales[at + tid];
        else vs_s[tid - AM_KEYS] = a.v_scales[at + tid - AM_KEYS];
        __syncthreads();
        // ---- scores of rows 4 rg .. + 3, keys kg + 16 j ----
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
        const float* qr = q_s + rg * 4 * hd;
        const __half* kr = k_s + kg * hs;
#pragma unroll 2
        for (int d = 0; d < hd; d += 4) {
            float4 q4[4], k4[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q4[i] = *reinterpret_cast<const float4*>(qr + i * hd + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) k4[j] = am_floats(kr + 16 * j * hs + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[i][j] = fmaf(q4[i].x, k4[j].x, s[i][j]); s[i][j] = fmaf(q4[i].y, k4[j].y, s[i][j]);
                    s[i][j] = fmaf(q4[i].z, k4[j].z, s[i][j]); s[i][j] = fmaf(q4[i].w, k4[j].w, s[i][j]);
                }
        }
        // ---- their weights ----
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float top = AQ_NEG;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = kg + 16 * j, p = j0 + key;
                const bool seen = p >= max(lo_w[i], lo) && p < min(hi_w[i], hi);
                s[i][j] = seen ? s[i][j] * ks_s[key] : AQ_NEG;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(m_r[i], top);
            const float m_use = top == AQ_NEG ? 0.0f : top, f = expf(m_r[i] - m_use);
            m_r[i] = top;
            l_r[i] *= f;
#pragma unroll
            for (int d = 0; d < 4 * NJ; ++d) acc[i][d] *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = kg + 16 * j, p = j0 + key;
                const bool seen = p >= max(lo_w[i], lo) && p < min(hi_w[i], hi);
                const float w = expf(s[i][j] - m_use);
                l_r[i] += w;
                s[i][j] = seen ? w * vs_s[key] : 0.0f;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) p_s[rg * AM_KEYS + kg + 16 * j] = make_float4(s[0][j], s[1][j], s[2][j], s[3][j]);
        __syncwarp();
        // ---- outputs: dimensions 4 kg + 64 j ----
#pragma unroll 4
        for (int key = 0; key < AM_KEYS; ++key) {
            const float4 w = p_s[rg * AM_KEYS + key];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
                if (64 * j + 64 <= hd || 64 * j + 4 * kg < hd) {
                    const float4 v = am_floats(v_s + key * hd + 64 * j + 4 * kg);
                    const float we[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[i][4 * j] = fmaf(we[i], v.x, acc[i][4 * j]);
                        acc[i][4 * j + 1] = fmaf(we[i], v.y, acc[i][4 * j + 1]);
                        acc[i][4 * j + 2] = fmaf(we[i], v.z, acc[i][4 * j + 2]);
                        acc[i][4 * j + 3] = fmaf(we[i], v.w, acc[i][4 * j + 3]);
                    }
                }
        }
        __syncwarp();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float l = l_r[i];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const int r = rg * 4 + i;
        if (r >= rows) continue;
        const size_t th = place_s[r];
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float* p = a.n_splits > 1 ? a.partial + (th * a.n_splits + split) * (hd + 2) : nullptr;
        if (p != nullptr && kg == 0) {
            // base-2 units, as the kernel of few rows leaves them
            p[0] = l != l ? INFINITY : m_r[i] * 1.4426950408889634f;
            p[1] = l;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int d = 64 * j + 4 * kg;
            if (d >= hd) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (p != nullptr) p[2 + d + e] = acc[i][4 * j + e];
                else ((T*)a.out)[th * hd + d + e] = from_f32<T>(acc[i][4 * j + e] * inv);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------
// The splits of one (token, head) joined in split order.  Partial results: maximum (base 2), sum, then
// the unnormalised output; a split without a visible key has a maximum of -infinity and no output.
// ------------------------------------------------------------------------------------------
template <typename T>
__global__ void attention_q8_merge_kernel(AttnQ8Args a) {
    pdl_prologue();
    const int n_splits = a.n_splits, hd = a.hd, G = a.n_heads / a.n_kv;
    extern __shared__ float mq_s[];                        // [n_splits] factors
    __shared__ float red_s[33];
    const size_t th = blockIdx.x;
    // tokens that no row has brought stay as they are
    const int token = blockIdx.x / a.n_heads, head = blockIdx.x - token * a.n_heads;
    bool held = false;
    for (int b = threadIdx.x; b < a.n_rows; b += blockDim.x) {
        const int from = a.cu_seqlens[b], to = a.cu_seqlens[b + 1];
        if (from >= 0 && from <= token && token < to && to <= a.n_tokens)
            held |= (long long)(token - from) * G + head % G < (long long)a.q_groups * a.block_rows;
    }
    if (!__syncthreads_or(held)) return;
    const float* p = a.partial + th * n_splits * (hd + 2);
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
        ((T*)a.out)[th * hd + d] = from_f32<T>(o * inv);
    }
}

// ---- host side ------------------------------------------------------------------------------
static bool aq_on_tensor_cores(int hd, int dtype) { return dtype == MF_DTYPE_BF16 && (hd == 64 || hd == 128); }

// blocks of the tensor-core kernel that an SM holds (its registers are cut for them)
static constexpr int aq_blocks_an_sm(int hd, int rows) {
    return hd == 128 ? (rows == 16 ? 3 : 2) : (rows <= 16 ? 4 : 3);
}

// matrix rows a block of the tensor-core kernel takes, from the most tokens a row brings
static int aq_block_rows(int max_row_tokens, int group) {
    const long long tiles = ((long long)max_row_tokens * group + 7) / 8;
    if (tiles <= 4) return (int)tiles * 8;
    const long long blocks = (tiles + 3) / 4;
    return (int)((tiles + blocks - 1) / blocks) * 8;
}

#define AQ_CLUSTER 8                           // most blocks of AQ_SPLIT's clusters
// How a call is shared out.  Tensor cores: AQ_WHOLE (splits 1), AQ_SPLIT (2, 4, 8) or AQ_SHARED (its blocks as a
// negative number); generic kernel: the splits of a row's keys.  `span`: the most positions the queries of
// one block can see, from a page's border on.  `floats`: the scratch it takes.
struct AqPlan {
    int rows, splits;
    long long floats;
};
static AqPlan aq_plan(int n_tokens, int n_rows, int max_row_tokens, int span, int n_heads, int n_kv, int hd, int dtype) {
    AqPlan p{};
    const int group = n_heads / n_kv;
    const int pages = span <= 0 ? 1 : (span + MF_PAGE - 1) / MF_PAGE, sms = mf_sm_count();
    const bool tensor = aq_on_tensor_cores(hd, dtype);
    auto items_of = [&](int rows) { return (long long)n_rows * n_kv * (((long long)max_row_tokens * group + rows - 1) / rows); };
    if (!tensor) {
        // 32 rows a block where that many are worth it and its pages are two blocks an SM at least.  us, 8 rows a block /
        // 32 (40 heads, 8 of keys, 128): 16 sequences of 3 tokens behind 2,000 346 / 244, 4 of 2 behind 600 31 / 33;
        // 38 of 36 behind 75 to 151 334 / 319; 4 of 1 to 3 behind 60 to 611 (14 and 2 heads of 64) 14.4 / 20.5; one of 512
        // behind none (28 and 4 of 128) 191 / 162; 8 of 16 behind 1,000 (8 and 2 of 256) 123 / 88; 39 of 8 behind 340 to
        // 680 (16 and 4 of 128) 145 / 160, the one loss found.
        p.rows = (long long)max_row_tokens * group > AM_LEAST && items_of(AM_ROWS) * pages >= 2LL * sms ? AM_ROWS : AG_ROWS;
        long long splits = 3LL * sms / items_of(p.rows);
        if (splits > pages) splits = pages;
        if (splits > AQ_MAX_SPLITS) splits = AQ_MAX_SPLITS;
        p.splits = splits < 1 ? 1 : (int)splits;
        p.floats = p.splits > 1 ? (long long)n_tokens * n_heads * p.splits * (hd + 2) : 0;
        return p;
    }
    p.rows = aq_block_rows(max_row_tokens, group);
    const long long items = items_of(p.rows);
    const int held = sms * aq_blocks_an_sm(hd, p.rows);
    int cluster = 1;
    while (2 * cluster <= AQ_CLUSTER && 2 * cluster * items <= held && 2 * cluster <= (pages + 3) / 4) cluster *= 2;
    // Clusters where they fill half of the GPU at least, or where a block has 12 pages at most; a block an item
    // where that is little.  us, whole / clusters / shared: 8 sequences at 2,000 positions (28 heads, 4 of
    // keys) - / 10.3 / 14.4, at 32,000 - / 48.0 / 53.0; 1 at 32,000 - / 39 / 20; 64 of 0 to 4,095 (14 and 2 heads of 64) -
    // / 16.4 / 26.6; 64 of 2,047 to 8,100 80 / - / 65; 128 of 500 23.1 / - / 27.4, of 2,000 64 / - / 55.
    if ((pages <= 12 || cluster > 1) && (pages <= 12 * cluster || 2LL * cluster * items >= held)) {
        p.splits = cluster;
        return p;
    }
    p.splits = -held;
    p.floats = (long long)aq_table_floats(held) + 2LL * held * (long long)aq_slot_floats(p.rows, hd);
    return p;
}

#define AQ_MAX_DEVICES 64
template <int HD, int FMT, int NT, int KT, int MODE, int STAGES, int MINB>
static int launch_mma_as(const AttnQ8Args& a, int items, int blocks, cudaStream_t stream) {
    constexpr int ring = AQ_WARPS * STAGES * KT * AqTile<HD>::STAGE, join = AQ_WARPS * 8 * NT * (HD + 4) * 4;
    constexpr int smem = ring > join ? ring : join;
    auto kernel = attention_q8_mma_kernel<HD, FMT, NT, KT, MODE, STAGES, MINB>;
    static bool opened[AQ_MAX_DEVICES] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= AQ_MAX_DEVICES || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return (int)e;
        if (dev >= 0 && dev < AQ_MAX_DEVICES) opened[dev] = true;
    }
    const dim3 grid = MODE == AQ_SHARED ? dim3(blocks) : MODE == AQ_WHOLE ? dim3(items, 1, a.n_rows) : dim3(a.n_splits, items, a.n_rows);
    if (MODE != AQ_SPLIT) {
        mf_launch(kernel, grid, dim3(AQ_WARPS * 32), smem, stream, a);
        if (int e = MF_LAUNCH_CHECK()) return e;
        if (MODE == AQ_SHARED && blocks > 1)
            mf_launch(attention_q8_join_kernel<HD, 8 * NT>, dim3(blocks - 1, 8 * NT), dim3(AQ_JOIN_WARPS * 32), 0, stream, a, blocks);
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
template <int HD, int FMT, int NT, int KT, int STAGES>
static int launch_mma(const AttnQ8Args& a, int items, int splits, cudaStream_t stream) {
    constexpr int minb = aq_blocks_an_sm(HD, 8 * NT);
    return splits < 0    ? launch_mma_as<HD, FMT, NT, KT, AQ_SHARED, STAGES, minb>(a, items, -splits, stream)
           : splits == 1 ? launch_mma_as<HD, FMT, NT, KT, AQ_WHOLE, STAGES, minb>(a, items, 0, stream)
                         : launch_mma_as<HD, FMT, NT, KT, AQ_SPLIT, STAGES, minb>(a, items, 0, stream);
}
static unsigned ag_by_row(int hd) { return (unsigned)((0x100000000ULL + hd / 4 - 1) / (hd / 4)); }
template <typename T, int FMT, int ND> static int launch_generic_as(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    const int smem = (AG_KEYS * (2 * a.hd + 4) + AG_ROWS * a.hd + 2 * AG_KEYS + AG_ROWS * AG_KEYS) * 4;
    constexpr int hd = 32 * ND, most = (AG_KEYS * (2 * hd + 4) + AG_ROWS * hd + 2 * AG_KEYS + AG_ROWS * AG_KEYS) * 4;
    static bool opened[AQ_MAX_DEVICES] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= AQ_MAX_DEVICES || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(attention_q8_generic_kernel<T, FMT, ND>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, most))
            return (int)e;
        if (dev >= 0 && dev < AQ_MAX_DEVICES) opened[dev] = true;
    }
    mf_launch(attention_q8_generic_kernel<T, FMT, ND>, grid, dim3(AG_WARPS * 32), smem, stream, a, ag_by_row(a.hd));
    return MF_LAUNCH_CHECK();
}
template <typename T, int FMT, int NJ> static int launch_rows_as(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    auto bytes = [](int hd) { return AM_KEYS * (2 * hd + 4) * 2 + (AM_ROWS * hd + 2 * AM_KEYS + AM_ROWS * AM_KEYS) * 4; };
    static bool opened[AQ_MAX_DEVICES] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= AQ_MAX_DEVICES || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(attention_q8_rows_kernel<T, FMT, NJ>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, bytes(64 * NJ)))
            return (int)e;
        if (dev >= 0 && dev < AQ_MAX_DEVICES) opened[dev] = true;
    }
    mf_launch(attention_q8_rows_kernel<T, FMT, NJ>, grid, dim3(128), (size_t)bytes(a.hd), stream, a, ag_by_row(a.hd));
    return MF_LAUNCH_CHECK();
}
template <typename T, int FMT> static int launch_generic(const AttnQ8Args& a, dim3 grid, cudaStream_t stream) {
    if (a.block_rows == AM_ROWS)
        return a.hd <= 64    ? launch_rows_as<T, FMT, 1>(a, grid, stream)
               : a.hd <= 128 ? launch_rows_as<T, FMT, 2>(a, grid, stream)
               : a.hd <= 192 ? launch_rows_as<T, FMT, 3>(a, grid, stream)
                             : launch_rows_as<T, FMT, 4>(a, grid, stream);
    return a.hd <= 32   ? launch_generic_as<T, FMT, 1>(a, grid, stream)
           : a.hd <= 64 ? launch_generic_as<T, FMT, 2>(a, grid, stream)
           : a.hd <= 128 ? launch_generic_as<T, FMT, 4>(a, grid, stream)
                         : launch_generic_as<T, FMT, 8>(a, grid, stream);
}

// The scratch of a call in floats; `kernels`: how many it launches.
extern "C" long long mf_attention_q8_plan(int n_tokens, int n_rows, int max_row_tokens, int span, int n_heads, int n_kv,
                                          int hd, int dtype, int* kernels) {
    *kernels = 1;
    if (n_rows <= 0 || max_row_tokens <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return 0;
    const AqPlan p = aq_plan(n_tokens, n_rows, max_row_tokens, span, n_heads, n_kv, hd, dtype);
    *kernels = p.floats > 0 ? 2 : 1;
    return p.floats;
}

// `partial` holds what mf_attention_q8_plan says for the same sizes, 16-byte aligned.
extern "C" int mf_attention_q8(const void* q, const void* k_codes, const void* v_codes, const float* k_scales,
                               const float* v_scales, const int* cu_seqlens, const int* seq_end, const int* page_table,
                               int table_stride, int ring, int n_pages, void* out, float* partial, int n_tokens,
                               int n_rows, int max_row_tokens, int span, int n_heads, int n_kv, int hd, int window,
                               float scale, int dtype, int fmt, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0 || n_rows <= 0 || max_row_tokens <= 0) return 0;
    if (hd % 16 != 0 || hd < 16 || hd > 256 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return MF_ERR_UNSUPPORTED;
    if ((dtype != MF_DTYPE_F32 && dtype != MF_DTYPE_BF16) || (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8))
        return MF_ERR_UNSUPPORTED;
    if (table_stride > (1 << 24)) return MF_ERR_UNSUPPORTED;         // (positions are 32 bits, with room to add)
    if (table_stride <= 0 || n_pages <= 0 || ring < 0 || ring % MF_PAGE != 0 || window < 0 || status == nullptr)
        return MF_ERR_ARGUMENT;
    AqPlan plan = aq_plan(n_tokens, n_rows, max_row_tokens, span, n_heads, n_kv, hd, dtype);
    if (plan.floats > 0 && (partial == nullptr || ((uintptr_t)partial & 15))) return MF_ERR_ARGUMENT;
    if (ring > 0 && (window <= 0 || max_row_tokens > ring - window + 1)) return MF_ERR_ARGUMENT;
    if (n_rows > 65535) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scales | (uintptr_t)v_scales |
         (uintptr_t)out) & 15)
        return MF_ERR_UNSUPPORTED;
    AttnQ8Args a{};
    a.q = q; a.k_codes = (const uint8_t*)k_codes; a.v_codes = (const uint8_t*)v_codes; a.k_scales = k_scales;
    a.v_scales = v_scales; a.cu_seqlens = cu_seqlens; a.seq_end = seq_end; a.page_table = page_table;
    a.table_stride = table_stride; a.ring = ring; a.n_pages = n_pages; a.out = out; a.partial = partial;
    a.n_tokens = n_tokens; a.n_rows = n_rows; a.n_heads = n_heads; a.n_kv = n_kv; a.hd = hd; a.window = window;
    a.n_splits = plan.splits < 0 ? 1 : plan.splits; a.scale = scale; a.status = status;
    const long long groups = ((long long)max_row_tokens * (n_heads / n_kv) + plan.rows - 1) / plan.rows;
    if (groups * n_kv > 0x7fffffffLL) return MF_ERR_UNSUPPORTED;
    a.q_groups = (int)groups;
    a.block_rows = plan.rows;
    a.max_end = ring > 0 ? 1 << 30 : table_stride * MF_PAGE;
    // (the pages of all items are counted in 32 bits)
    const long long row_pages = ring > 0 ? ((long long)window + n_tokens) / MF_PAGE + 3 : table_stride;
    if (plan.splits < 0 && row_pages * groups * n_kv * n_rows > 0x7fffffffLL) plan.splits = 1;
    const int items = (int)(groups * n_kv), n_splits = a.n_splits;
    const dim3 grid(items, n_splits, n_rows);
    int e;
    if (aq_on_tensor_cores(hd, dtype)) {
#define AQ_GO(HD, NT, KT, STAGES)                                                                 \
    (fmt == MF_Q8_E4M3 ? launch_mma<HD, MF_Q8_E4M3, NT, KT, STAGES>(a, items, plan.splits, stream) \
                       : launch_mma<HD, MF_Q8_INT8, NT, KT, STAGES>(a, items, plan.splits, stream))
        const int nt = plan.rows / 8;
        if (hd == 128) return nt == 1 ? AQ_GO(128, 1, 2, 3) : nt == 2 ? AQ_GO(128, 2, 1, 4) : nt == 3 ? AQ_GO(128, 3, 1, 4) : AQ_GO(128, 4, 1, 4);
        return nt == 1 ? AQ_GO(64, 1, 2, 3) : nt == 2 ? AQ_GO(64, 2, 1, 6) : nt == 3 ? AQ_GO(64, 3, 1, 6) : AQ_GO(64, 4, 1, 6);
#undef AQ_GO
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
                  (size_t)n_splits * 4, stream, a);
    else
        mf_launch(attention_q8_merge_kernel<__nv_bfloat16>, dim3((unsigned)(n_tokens * n_heads)), dim3(threads),
                  (size_t)n_splits * 4, stream, a);
    return MF_LAUNCH_CHECK();
}
