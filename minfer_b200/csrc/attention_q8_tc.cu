// Attention of portions (many new tokens a row) over a paged cache of 8-bit keys and values, bfloat16
// queries, head size 64 or 128, on tcgen05.  The formula is that of attention_q8.cu:
//
//   o_i = sum_j p_ij vs_j vc_j / sum_j p_ij,   p_ij = exp(scale q_i . kc_j ks_j - max)
//
// Keys and values go to the tensor cores as halves, each brought below 2^15 by one power of two of its 128
// positions; queries are exact halves by a power of two of their vector; probabilities are rounded to halves, too:
// keys, values and probabilities are off by 2^-11 each, where bfloat16 is by 2^-8.  (Codes multiplied as they are,
// exactly, with the scales applied to scores and probabilities: a row's 128 keys need 384 scales out of shared
// memory, 3,072 of the 5,200 clocks that a tile then took; this way it takes 3,800.)  Where scales of 128 positions
// are more than 2^QT_APART apart (a half's range; a token may not see the one that is far above the others), every
// position has a power of two of its own, which its scores and probabilities are multiplied by.
//
// Three launches:
//   unpack   what the rows' tokens can see, position behind position (a window over a ring becomes a
//            stretch), and the queries, as halves
//   attend   a block an SM: items (row, 256 tokens, head), each some tiles of 128 keys, are laid end to
//            end and dealt out evenly, wherever one item ends and the next begins.  512 tokens of 40 heads
//            are 80 items, which leave 68 of 148 SMs idle where a block takes whole ones.
//   join     the items that several blocks have worked on
//
// attend is built like the prompts' kernel: a warp issues TMA copies, one the products, and a warpgroup for
// each of two tiles of 128 queries takes a row of scores a thread out of tensor memory, forms the
// softmax and puts probabilities back as the A operand of the second product.  Tensor memory: S0 S1 O0 O1.
//
// The reference of a row's exponentials goes by what is rounded: 2^(s_j - m) times the power of two of the tile's
// values, 2^6 at the largest and up to 2^14 before the reference moves; the sum of 2^(s_j - m) is float32.
//
// A scale of NaN marks a vector that was not finite: such a key is NaN, its score too for the tokens that see it,
// and it is masked for the others; a value's mark is moved to its key, so that zero times NaN is never formed.
#include "prefill_tc.cuh"
#include "q8.cuh"

#include <type_traits>

#define QT_Q 128              // queries a tile
#define QT_ITEM 256           // queries an item: two tiles
#define QT_KEYS 128           // keys a tile
#define QT_THREADS 384        // a warpgroup for copies and products, one for each query tile
#define QT_BELOW 6.0f         // the reference is put 2^6 below the largest weight, and moves when one passes it by 2^14
#define QT_ROOM 14.0f
#define QT_LEAST 4            // least tiles a block takes
#define QT_APART 16           // binary orders that scales of a tile share a power of two over
#define QT_WIDE 1000.0f       // in place of a tile's exponents: its positions have their own
#define QT_LEAST_VALUE (-60)  // values' power of two at least (sums of 2^(s_j - m) stay in float32's range)

struct QtArgs {
    const __nv_bfloat16* q;
    const uint8_t* k_codes;
    const uint8_t* v_codes;
    const float* k_scales;
    const float* v_scales;
    const int* cu_seqlens;
    const int* seq_end;
    const int* page_table;
    int table_stride, ring, n_pages;
    int max_end;              // positions a row may have
    int stretch;              // positions a row has room for in the scratch, a multiple of 128
    __nv_bfloat16* out;
    int n_tokens, n_rows, n_heads, n_kv, window, with_q;
    float scale;
    unsigned* status;
    // scratch
    __half* k16;              // [rows][n_kv][stretch][HD]
    __half* v16;
    float2* powers;           // [rows][n_kv][stretch / 128]: the exponents of keys and values, or QT_WIDE
    float* own;               // [rows][n_kv][stretch / 128][2][128]: the positions' powers of two, keys and values
    __half* q16;              // [tokens][n_heads][HD]
    float* factor;            // [tokens][n_heads]: scores in powers of two of 2
    int4* first;              // [blocks]: row, item of the row, tile of it, tiles a block
    float* slots;             // [blocks][2][HD / 4][256][4] outputs, [256] maxima, [256] sums
};

// A row's tokens (brought inside what there is), the position its stretch begins with and the first that is seen.
struct QtRow {
    int tok0, count, end, base, seen;
};
__device__ __forceinline__ QtRow qt_row(const QtArgs& a, int b) {
    QtRow r;
    const int from = a.cu_seqlens[b], to = a.cu_seqlens[b + 1], e = a.seq_end[b];
    r.tok0 = from;
    r.count = from >= 0 && from <= to && to <= a.n_tokens ? to - from : 0;
    r.end = min(max(e, 0), a.max_end);
    r.seen = a.window > 0 ? max(0, r.end - r.count - a.window + 1) : 0;
    r.base = r.seen & ~(QT_KEYS - 1);
    return r;
}
// The key tiles of the row's queries q0 .. q0 + 255: [lo, hi), one at least (a query that sees nothing has
// zeros to write).
__device__ __forceinline__ void qt_tiles(const QtArgs& a, const QtRow& r, int q0, int* lo, int* n) {
    const int start = r.end - r.count, last = start + min(q0 + QT_ITEM, r.count) - 1;
    const int from = a.window > 0 ? max(0, start + q0 - a.window + 1) : 0, most = a.stretch / QT_KEYS;
    *lo = min(max(0, from - r.base) / QT_KEYS, most - 1);
    const int hi = last < r.base ? 0 : min(most, (last - r.base) / QT_KEYS + 1);
    *n = max(1, hi - *lo);
}
__device__ __forceinline__ int qt_items(const QtRow& r) { return (r.count + QT_ITEM - 1) / QT_ITEM; }

// ------------------------------------------------------------------------------------------
// unpack: bound by bytes, 1 read and 2 written a code.  A block takes 128 positions of one key/value head, K or V,
// a thread's unit 8 codes (whole lines a warp); the blocks behind them 32 query vectors each, a warp four.
// ------------------------------------------------------------------------------------------
#define QU_THREADS 256
#define QU_VECTORS 32
template <int FMT, int HD>
__global__ void __launch_bounds__(QU_THREADS) q8_unpack_kernel(QtArgs a, int n_tiles_all) {
    pdl_launch_dependents();
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= n_tiles_all) {
        // ---- queries ----
        constexpr int PER = HD / 32;                       // elements a lane
        const int warp = tid >> 5, lane = tid & 31;
        const long long first = (long long)(blockIdx.x - n_tiles_all) * QU_VECTORS + warp * 4;
        const long long all = (long long)a.n_tokens * a.n_heads;
        pdl_wait();
        uint32_t w[4][PER / 2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long at = min(first + i, all - 1) * HD + lane * PER;
            if constexpr (PER == 4) {
                const uint2 x = *reinterpret_cast<const uint2*>(a.q + at);
                w[i][0] = x.x; w[i][1] = x.y;
            } else {
                w[i][0] = *reinterpret_cast<const uint32_t*>(a.q + at);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned top = 0;
#pragma unroll
            for (int j = 0; j < PER / 2; ++j) top = max(top, max(w[i][j] & 0x7fffu, (w[i][j] >> 16) & 0x7fffu));
            top = __reduce_max_sync(0xffffffffu, top);
            // 2^(14 - exponent), from the exponent field (numbers below the normal range: 2^100)
            const bool bad = top >= 0x7f80u;
            const int field = (int)(top >> 7), power = field == 0 ? 100 : min(141 - field, 100);
            // (a negative scale goes on the queries, and so does 0: factors are above 0, which keeps masked
            // scores at -infinity)
            float up = __int_as_float((power + 127) << 23);
            if (a.scale < 0.0f) up = -up;
            if (a.scale == 0.0f || bad) up = 0.0f;
            uint32_t h[PER / 2];
#pragma unroll
            for (int j = 0; j < PER / 2; ++j) {
                const float lo = bad ? 0.0f : __uint_as_float(w[i][j] << 16) * up;
                const float hi = bad ? 0.0f : __uint_as_float(w[i][j] & 0xffff0000u) * up;
                const __half2 x = __floats2half2_rn(lo, hi);
                h[j] = *reinterpret_cast<const uint32_t*>(&x);
            }
            if (first + i >= all) continue;
            __half* to = a.q16 + (first + i) * HD + lane * PER;
            if constexpr (PER == 4) *reinterpret_cast<uint2*>(to) = make_uint2(h[0], h[1]);
            else *reinterpret_cast<uint32_t*>(to) = h[0];
            if (lane == 0) {
                const float by = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.4426950408889634f * __int_as_float((127 - power) << 23);
                a.factor[first + i] = bad ? __int_as_float(0x7fc00000) : fmaxf(by, 1.2e-38f);
            }
        }
        return;
    }
    // ---- 128 positions of a row ----
    const int tiles = a.stretch / QT_KEYS;
    int u = blockIdx.x;
    const bool is_v = u & 1;
    u >>= 1;
    const int hk = u % a.n_kv;
    u /= a.n_kv;
    const int i = u % tiles, b = u / tiles;
    const QtRow r = qt_row(a, b);
    const int p0 = r.base + i * QT_KEYS;
    // (a first tile that holds no position is read)
    if (r.count == 0 || p0 >= max(r.end, r.base + 1)) { pdl_wait(); return; }
    if (tid == 0 && i == 0 && hk == 0 && !is_v && a.seq_end[b] > a.max_end) atomicOr(a.status, MF_STATUS_BAD_POSITION);
    const int n0 = max(0, r.seen - p0), n1 = min(QT_KEYS, r.end - p0);       // places [n0, n1) are seen
    long long from[2];                                                       // the two pages' vectors; -1: none
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int p = p0 + h * MF_PAGE, index = (a.ring > 0 ? p % a.ring : p) >> 6;
        const bool seen = n1 > h * MF_PAGE && n0 < (h + 1) * MF_PAGE && n1 > n0;
        const int page = seen && index < a.table_stride ? a.page_table[(size_t)b * a.table_stride + index] : -1;
        const bool there = page >= 0 && page < a.n_pages;
        if (seen && !there && tid == 0 && hk == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
        from[h] = there ? ((long long)page * a.n_kv + hk) * MF_PAGE : -1;
    }
    __shared__ float scale_s[QT_KEYS];
    __shared__ unsigned most_s[QT_KEYS / 32], least_s[QT_KEYS / 32];
    pdl_wait();
    const uint8_t* codes = is_v ? a.v_codes : a.k_codes;
    constexpr int EACH = QT_KEYS * HD / 8 / QU_THREADS;
    uint2 w[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        // (a page is half of a tile's units)
        const int unit = tid + (j % (EACH / 2)) * QU_THREADS, place = unit / (HD / 8) + (j / (EACH / 2)) * MF_PAGE;
        const long long at = from[j / (EACH / 2)];
        const bool held = at >= 0 && place >= n0 && place < n1;              // (what other places hold is anybody's)
        w[j] = held ? *reinterpret_cast<const uint2*>(codes + at * HD + unit * 8) : make_uint2(0, 0);
    }
    if (tid < QT_KEYS) {
        const long long at = tid < MF_PAGE ? from[0] : from[1];
        const bool held = at >= 0 && tid >= n0 && tid < n1;
        const float ks = held ? a.k_scales[at + tid % MF_PAGE] : 0.0f, vs = held ? a.v_scales[at + tid % MF_PAGE] : 0.0f;
        float x = is_v ? vs : ks;
        if (is_v && vs != vs) x = 0.0f;
        if (!is_v && vs != vs) x = vs;
        scale_s[tid] = x;
        const unsigned bits = x == x ? __float_as_uint(fabsf(x)) : 0u;
        const unsigned most = __reduce_max_sync(0xffffffffu, bits);
        const unsigned least = __reduce_min_sync(0xffffffffu, bits == 0 ? 0x7f800000u : bits);
        if ((tid & 31) == 0) { most_s[tid >> 5] = most; least_s[tid >> 5] = least; }
    }
    __syncthreads();
    // the largest scale (or every one) to 2^5 .. 2^6, times a code below 2^15
    auto power_of = [&](unsigned bits) {
        return bits == 0 ? 0 : min(max((int)(bits >> 23) - 127 - 5, is_v ? QT_LEAST_VALUE : -120), 120);
    };
    const unsigned most = max(max(most_s[0], most_s[1]), max(most_s[2], most_s[3]));
    const unsigned least = min(min(least_s[0], least_s[1]), min(least_s[2], least_s[3]));
    const int power = power_of(most);
    const bool wide = power - power_of(min(least, most)) > QT_APART;
    const long long tile = ((long long)b * a.n_kv + hk) * tiles + i;
    if (tid == 0) (is_v ? a.powers[tile].y : a.powers[tile].x) = wide ? QT_WIDE : (float)power;
    if (tid < QT_KEYS) {
        const float x = scale_s[tid];
        const int mine = wide ? power_of(x == x ? __float_as_uint(fabsf(x)) : 0u) : power;
        a.own[tile * (2 * QT_KEYS) + (is_v ? QT_KEYS : 0) + tid] = __int_as_float((127 + mine) << 23);
        scale_s[tid] = x * __int_as_float((127 - mine) << 23);
    }
    __syncthreads();
    __half* out = (is_v ? a.v16 : a.k16) + tile * (QT_KEYS * HD);
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int unit = tid + j * QU_THREADS;
        const float by = scale_s[unit / (HD / 8)];
        float v[8];
        q8_floats<FMT>(w[j].x, v);
        q8_floats<FMT>(w[j].y, v + 4);
        uint32_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const __half2 x = __floats2half2_rn(v[2 * e] * by, v[2 * e + 1] * by);
            h[e] = *reinterpret_cast<const uint32_t*>(&x);
        }
        *reinterpret_cast<uint4*>(out + unit * 8) = make_uint4(h[0], h[1], h[2], h[3]);
    }
}

// ------------------------------------------------------------------------------------------
// attend
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t qt_pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint64_t qt_pair(const uint32_t* r) {
    return fa_pack2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
constexpr __host__ __device__ size_t qt_slot_floats(int hd) { return (size_t)QT_ITEM * (hd + 2); }
__device__ __forceinline__ int qt_share(int units, int blocks) { return max(QT_LEAST, (units + blocks - 1) / blocks); }

// A block's way through its tiles: part [off, off + part) of an item's n tiles, the first of them `lo`.
struct QtWalk {
    QtRow row;
    int b, group, head, lo, n, off, part, todo;
    __device__ __forceinline__ void look(const QtArgs& a) {
        qt_tiles(a, row, group * QT_ITEM, &lo, &n);
        part = min(todo, n - off);
    }
    // on to the next item; false: nothing is left
    __device__ __forceinline__ bool next(const QtArgs& a) {
        todo -= part;
        if (todo <= 0) return false;
        off = 0;
        if (++head == a.n_heads) {
            head = 0;
            if (++group == qt_items(row)) {
                group = 0;
                do row = qt_row(a, ++b); while (row.count == 0);
            }
        }
        look(a);
        return true;
    }
};

template <int HD>
__global__ void __launch_bounds__(QT_THREADS, 1)
attention_q8_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                       const __grid_constant__ CUtensorMap map_v, const QtArgs a) {
    pdl_launch_dependents();
    constexpr int NB = HD / 64;                         // 64-column blocks a row
    constexpr int BLOCK = 128 * 128;                    // bytes of [128 rows][64 columns]
    constexpr int T_BYTES = NB * BLOCK;
    constexpr int TM_S = 0, TM_O = 256;                 // tensor memory columns; tile t: + 128 t
    extern __shared__ uint8_t qt_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)qt_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = smem;                                // [2 query tiles][NB][128][64]
    uint8_t* k_s = q_s + 2 * T_BYTES;                   // [2 stages]
    uint8_t* v_s = k_s + 2 * T_BYTES;                   // [2 stages]
    uint64_t* bars = (uint64_t*)(v_s + 2 * T_BYTES);
    uint64_t* q_full = bars;
    uint64_t* q_empty = bars + 1;
    uint64_t* k_full = bars + 2;                        // [2 stages] each
    uint64_t* k_empty = bars + 4;
    uint64_t* v_full = bars + 6;
    uint64_t* v_empty = bars + 8;
    uint64_t* s_full = bars + 10;                       // [2 query tiles] each
    uint64_t* p_half = bars + 12;                       // 128 arrivals: the first 64 keys' weights
    uint64_t* p_full = bars + 14;                       // 128 arrivals
    uint64_t* o_done = bars + 16;
    uint32_t* tmem_slot = (uint32_t*)(bars + 18);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    __shared__ int scan_s[QT_THREADS / 32], at_s[2];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // ---- which tiles of which items: the tiles of all rows, and the row that the block's first one belongs to ----
    int units = 0, before = 0, share = 0, begin = 0, todo = 0;
    for (int b0 = 0; b0 < a.n_rows;) {
        int mine = 0;
        if (b0 + tid < a.n_rows) {
            const QtRow r = qt_row(a, b0 + tid);
            for (int g = 0; g < qt_items(r); ++g) {
                int lo, n;
                qt_tiles(a, r, g * QT_ITEM, &lo, &n);
                mine += n * a.n_heads;
            }
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
        for (int w = 0; w < QT_THREADS / 32; ++w) {
            if (w < warp) upto += scan_s[w];
            all += scan_s[w];
        }
        const bool known = share > 0;                   // (the second time through)
        if (!known) units += all;
        const bool done = !known && b0 + QT_THREADS >= a.n_rows;
        if (done) {
            share = qt_share(units, gridDim.x);
            begin = blockIdx.x * share;
            todo = min(share, units - begin);
        }
        if (known || a.n_rows <= QT_THREADS) {
            const int from = before + upto - mine;
            if (mine > 0 && from <= begin && begin < from + mine) { at_s[0] = b0 + tid; at_s[1] = from; }
            before += all;
        }
        b0 += QT_THREADS;
        if (done && a.n_rows > QT_THREADS && todo > 0) b0 = 0;       // once more, with the block's tile known
    }
    __syncthreads();
    if (todo <= 0) {
        pdl_wait();
        if (tid == 0) a.first[blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
    }
    QtWalk at;
    at.b = at_s[0];
    at.row = qt_row(a, at.b);
    at.todo = todo;
    {
        int rest = begin - at_s[1];
        for (at.group = 0;; ++at.group) {
            qt_tiles(a, at.row, at.group * QT_ITEM, &at.lo, &at.n);
            if (rest < at.n * a.n_heads || at.group + 1 >= qt_items(at.row)) break;
            rest -= at.n * a.n_heads;
        }
        at.head = rest / at.n;
        at.off = rest - at.head * at.n;
        at.part = min(todo, at.n - at.off);
    }

    if (tid == 0) {
        fa_bar_init(fa_smem(q_full), 1);
        fa_bar_init(fa_smem(q_empty), 1);
        for (int i = 0; i < 2; ++i) {
            fa_bar_init(fa_smem(&k_full[i]), 1);
            fa_bar_init(fa_smem(&k_empty[i]), 1);
            fa_bar_init(fa_smem(&v_full[i]), 1);
            fa_bar_init(fa_smem(&v_empty[i]), 1);
            fa_bar_init(fa_smem(&s_full[i]), 1);
            fa_bar_init(fa_smem(&p_half[i]), 128);
            fa_bar_init(fa_smem(&p_full[i]), 128);
            fa_bar_init(fa_smem(&o_done[i]), 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    pdl_wait();
    if (tid == 0) a.first[blockIdx.x] = make_int4(at.b, at.group * a.n_heads + at.head, at.off, share);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(fa_smem(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fa_fence_before();
    __syncthreads();
    fa_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Registers: compiled for 168 a thread, 64,512 in all; the first warpgroup gives half of its share to the other
    // two: 128 * 88 + 256 * 208 = 64,512.  (At 56 its two walks through the items spill: 3 % slower.)
    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == 0 && elect_one()) {
        // ---- TMA producer: `i` counts the block's tiles, `s` its items ----
        int i = 0;
        bool ok = true;
        for (int s = 0; ok; ++s) {
            const int q0 = at.group * QT_ITEM, hk = at.head / (a.n_heads / a.n_kv);
            const int tiles = q0 + QT_Q < at.row.count ? 2 : 1;
            if (s > 0 && !fa_wait(fa_smem(q_empty), (uint32_t)((s - 1) & 1), abort_flag)) break;
            fa_expect_tx(fa_smem(q_full), tiles * T_BYTES);
            for (int t = 0; t < tiles; ++t)
                for (int c = 0; c < NB; ++c)
                    fa_tma(fa_smem(q_s + t * T_BYTES + c * BLOCK), &map_q, at.head * HD + 64 * c,
                           at.row.tok0 + q0 + t * QT_Q, fa_smem(q_full));
            const int tile0 = (at.b * a.n_kv + hk) * (a.stretch / QT_KEYS) + at.lo + at.off;
            for (int j = 0; j < at.part; ++j, ++i) {
                const int st = i & 1;
                const uint32_t free_parity = (uint32_t)((i >> 1) & 1) ^ 1u;
                if (!fa_wait(fa_smem(&k_empty[st]), free_parity, abort_flag)) { ok = false; break; }
                fa_expect_tx(fa_smem(&k_full[st]), T_BYTES);
                for (int c = 0; c < NB; ++c)
                    fa_tma(fa_smem(k_s + st * T_BYTES + c * BLOCK), &map_k, 64 * c, (tile0 + j) * QT_KEYS, fa_smem(&k_full[st]));
                if (!fa_wait(fa_smem(&v_empty[st]), free_parity, abort_flag)) { ok = false; break; }
                fa_expect_tx(fa_smem(&v_full[st]), T_BYTES);
                for (int c = 0; c < NB; ++c)
                    fa_tma(fa_smem(v_s + st * T_BYTES + c * BLOCK), &map_v, 64 * c, (tile0 + j) * QT_KEYS, fa_smem(&v_full[st]));
            }
            if (!ok || !at.next(a)) break;
        }
      } else if (warp == 1 && elect_one()) {
        // ---- MMA issuer: halves into float32.  S: M = 128 queries, N = 128 keys, both operands K-major ----
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(QT_KEYS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        // O: M = 128 queries, N = HD, A from tensor memory, B MN-major
        constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        auto issue_qk = [&](int t, int st) {
            const uint32_t q_addr = fa_smem(q_s + t * T_BYTES), k_addr = fa_smem(k_s + st * T_BYTES);
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                const uint32_t off = (uint32_t)((ks >> 2) * BLOCK + (ks & 3) * 32);
                fa_mma_ss(tmem + (uint32_t)(TM_S + t * 128), fa_desc_kmajor(q_addr + off), fa_desc_kmajor(k_addr + off),
                          idesc_s, ks > 0 ? 1u : 0u);
            }
            fa_commit(fa_smem(&s_full[t]));
        };
        int i = 0, done[2] = {0, 0};                     // tiles begun; products P V issued for each query tile
        bool ok = true;
        for (int s = 0; ok; ++s) {
            const int tiles = at.group * QT_ITEM + QT_Q < at.row.count ? 2 : 1;
            ok = fa_wait(fa_smem(q_full), (uint32_t)(s & 1), abort_flag) &&
                 fa_wait(fa_smem(&k_full[i & 1]), (uint32_t)((i >> 1) & 1), abort_flag);
            if (!ok) break;
            fa_fence_after();
            for (int t = 0; t < tiles; ++t) issue_qk(t, i & 1);
            fa_commit(fa_smem(&k_empty[i & 1]));
            if (at.part == 1) fa_commit(fa_smem(q_empty));
            for (int j = 0; j < at.part && ok; ++j, ++i) {
                const bool next = j + 1 < at.part;
                ok = fa_wait(fa_smem(&v_full[i & 1]), (uint32_t)((i >> 1) & 1), abort_flag);
                if (ok && next) ok = fa_wait(fa_smem(&k_full[(i + 1) & 1]), (uint32_t)(((i + 1) >> 1) & 1), abort_flag);
                if (!ok) break;
                fa_fence_after();
                const uint32_t v_addr = fa_smem(v_s + (i & 1) * T_BYTES);
                for (int t = 0; t < tiles; ++t) {
#pragma unroll
                    for (int ks = 0; ks < QT_KEYS / 16; ++ks) {
                        // (the first half of the keys is multiplied while the others' exponentials are formed)
                        if (ks % (QT_KEYS / 32) == 0) {
                            ok = fa_wait(fa_smem(ks == 0 ? &p_half[t] : &p_full[t]), (uint32_t)(done[t] & 1), abort_flag);
                            if (!ok) break;
                            fa_fence_after();
                        }
                        fa_mma_ts(tmem + (uint32_t)(TM_O + t * 128), tmem + (uint32_t)(TM_S + t * 128 + ks * 8),
                                  fa_desc_mnmajor(v_addr + (uint32_t)(ks * 16 * 128), BLOCK), idesc_o,
                                  (j > 0 || ks > 0) ? 1u : 0u);
                    }
                    if (!ok) break;
                    ++done[t];
                    if (next) issue_qk(t, (i + 1) & 1);
                    else fa_commit(fa_smem(&o_done[t]));
                }
                if (!ok) break;
                fa_commit(fa_smem(&v_empty[i & 1]));
                if (next) fa_commit(fa_smem(&k_empty[(i + 1) & 1]));
                if (j + 2 == at.part) fa_commit(fa_smem(q_empty));   // the item's last scores have been asked for
            }
            if (!ok || !at.next(a)) break;
        }
      }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- softmax: four warps for each query tile, one thread a query row (two threads, which tell each other
        // their halves' maxima, take 4,300 clocks a tile where this takes 3,800) ----
        const int t = (warp - 4) >> 2;
        const int quarter = warp & 3;                    // the 32 lanes of tensor memory this warp may touch
        const int trow = quarter * 32 + lane;            // row of the tile
        const uint32_t lane_addr = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t s_addr = lane_addr + (uint32_t)(TM_S + t * 128);
        const uint32_t o_addr = lane_addr + (uint32_t)(TM_O + t * 128);
        int mine = 0, items = 0;                         // tiles and items of this query tile
        // (a warp gives up as one: what follows wants all its lanes)
        auto wait = [&](uint64_t* bar, int phase) {
            return (bool)__all_sync(0xffffffffu, fa_wait(fa_smem(bar), (uint32_t)(phase & 1), abort_flag));
        };
        bool ok = true;
        for (;;) {
            const int q0t = at.group * QT_ITEM + t * QT_Q, qrow = q0t + trow;
            const bool part_of = q0t < at.row.count;     // (the second tile may lie behind the row's tokens)
            const int start = at.row.end - at.row.count, wpos = start + q0t + quarter * 32;
            const bool real = qrow < at.row.count;
            const float by = real ? a.factor[(long long)(at.row.tok0 + qrow) * a.n_heads + at.head] : 1.0f;
            // the reference, the sum, and an exponent that outputs are to be multiplied by (0 unless scores are beyond
            // 2^20, where a reference does not tell a value's exponent from a rounding)
            float m = -INFINITY, l = 0.0f, r = 0.0f;
            const long long tile0 = (at.b * a.n_kv + at.head / (a.n_heads / a.n_kv)) * (long long)(a.stretch / QT_KEYS) + at.lo + at.off;
            const float2* powers = a.powers + tile0;
            float2 power = part_of ? powers[0] : make_float2(0.0f, 0.0f);
            for (int j = 0; part_of && j < at.part; ++j) {
                // (factors above 0 keep masked scores at -infinity)
                bool apart = power.x == QT_WIDE || power.y == QT_WIDE;
                float by_tile = fminf(fmaxf(by * __int_as_float((127 + (int)power.x) << 23), 1.2e-38f), 3e38f), values = power.y;
                if (apart) by_tile = 1.0f;
                const float4* own = reinterpret_cast<const float4*>(a.own + (tile0 + j) * (2 * QT_KEYS));
                if (j + 1 < at.part) power = powers[j + 1];
                // S of this key tile is complete, and with it every earlier product of this query tile
                if (!(ok = wait(&s_full[t], mine++))) break;
                fa_fence_after();
                const int key0 = at.row.base + (at.lo + at.off + j) * QT_KEYS;
                const bool need_mask = key0 + QT_KEYS - 1 > wpos || (a.window > 0 && key0 < wpos + 31 - a.window + 1);
                uint32_t sr[QT_KEYS];
#pragma unroll
                for (int c0 = 0; c0 < QT_KEYS; c0 += 32) fa_ld32(s_addr + (uint32_t)c0, sr + c0);
                fa_wait_ld();
                if (need_mask) {
                    const int qpos = start + qrow;
                    const int first = a.window > 0 ? qpos - a.window + 1 - key0 : 0, last = qpos - key0;
#pragma unroll
                    for (int e = 0; e < QT_KEYS; ++e)
                        if (e > last || e < first) sr[e] = 0xff800000u;              // -infinity
                }
                // the largest score, with four chains of three-input maxima
                float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
                for (int e = 0; e < QT_KEYS; e += 8) {
                    mx0 = fa_max3(mx0, __uint_as_float(sr[e]), __uint_as_float(sr[e + 1]));
                    mx1 = fa_max3(mx1, __uint_as_float(sr[e + 2]), __uint_as_float(sr[e + 3]));
                    mx2 = fa_max3(mx2, __uint_as_float(sr[e + 4]), __uint_as_float(sr[e + 5]));
                    mx3 = fa_max3(mx3, __uint_as_float(sr[e + 6]), __uint_as_float(sr[e + 7]));
                }
                float m_tile = fmaf(fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)), by_tile, values);
                // (differences of scores beyond 2^20 are to be those of rounded products: a fused one is off by what the
                // reference was rounded by)
                apart = apart || (fabsf(m_tile) > 1048576.0f && m_tile > -INFINITY);
                float r_new = r, m_far = -INFINITY;
                if (apart) {
                    // every position by its own powers of two; the largest weight: a score and its value's exponent
                    float top = -INFINITY, v_top = -INFINITY;
                    m_tile = -INFINITY;
#pragma unroll
                    for (int e = 0; e < QT_KEYS; e += 4) {
                        const float4 k = own[e >> 2], v = own[(QT_KEYS + e) >> 2];
                        const float ke[4] = {k.x, k.y, k.z, k.w}, ve[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const float x = __fmul_rn(__uint_as_float(sr[e + h]) * ke[h], by);
                            const float power = (float)((__float_as_int(ve[h]) >> 23) - 127);
                            sr[e + h] = __float_as_uint(x);
                            top = fmaxf(top, x);
                            if (x > -INFINITY) v_top = fmaxf(v_top, power);
                            m_tile = fmaxf(m_tile, x + power);
                        }
                    }
                    by_tile = 1.0f;
                    values = 0.0f;
                    if (fabsf(top) > 1048576.0f && top > -INFINITY) {
                        const bool above = m == -INFINITY || top - m > 256.0f;      // (what came before weighs nothing)
                        r_new = above ? v_top : fmaxf(r, v_top);
                        m_far = above ? top : fmaxf(m, top);
                    }
                }
                if (r != 0.0f && m_far == -INFINITY && m_tile - r - m > 256.0f) r_new = 0.0f;
                const float m_here = m_tile - r_new;
                const bool jump = m_far > -INFINITY ? m_far != m || r_new != r
                                  : m == -INFINITY  ? m_here > -INFINITY
                                                    : m_here - m > QT_ROOM;
                const float m_new = !jump ? m : m_far > -INFINITY ? m_far : m_here - QT_BELOW;
                const float m_off = m_new == -INFINITY ? 0.0f : m_new;
                __syncwarp();
                // the output so far is rescaled only if the reference moved for some row of this warp
                if (j > 0 && __any_sync(0xffffffffu, jump)) {
                    const float corr = jump ? (m == -INFINITY ? 0.0f : exp2f((m - m_off) + (r - r_new))) : 1.0f;
                    l *= jump ? (m == -INFINITY ? 0.0f : exp2f(m - m_off)) : 1.0f;
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 32) {
                        uint32_t w[32];
                        fa_ld32(o_addr + (uint32_t)c0, w);
                        fa_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * corr);
                        fa_st32(o_addr + (uint32_t)c0, w);
                    }
                }
                m = m_new;
                r = r_new;
                // weights 2^(s - m) times the values' power of two, their sum, and as halves into the first 64 columns
                // of S
                uint64_t l01 = 0, l23 = 0;               // four zeros
                const float off = apart ? -m_off : values - r - m_off;
                const uint64_t by2 = fa_pack2(by_tile, by_tile), off2 = fa_pack2(off, off);
                auto weigh = [&](auto apart_tag) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t pk[QT_KEYS / 4];
#pragma unroll
                        for (int g = 0; g < QT_KEYS / 2; g += 4) {
                            const int e = h * (QT_KEYS / 2) + g;
                            float x0, x1, x2, x3;
                            fa_unpack2(fa_fma2(qt_pair(sr + e), by2, off2), x0, x1);
                            fa_unpack2(fa_fma2(qt_pair(sr + e + 2), by2, off2), x2, x3);
                            asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x0));
                            asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x1));
                            asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x2));
                            asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(x3));
                            l01 = fa_add2(l01, fa_pack2(x0, x1));
                            l23 = fa_add2(l23, fa_pack2(x2, x3));
                            if constexpr (decltype(apart_tag)::value) {
                                const float4 v = own[(QT_KEYS + e) >> 2];
                                const float down_r = exp2f(-r);
                                x0 *= apart ? v.x * down_r : 1.0f; x1 *= apart ? v.y * down_r : 1.0f;
                                x2 *= apart ? v.z * down_r : 1.0f; x3 *= apart ? v.w * down_r : 1.0f;
                            }
                            pk[g >> 1] = qt_pack(x0, x1);
                            pk[(g >> 1) + 1] = qt_pack(x2, x3);
                        }
                        fa_st32(s_addr + (uint32_t)(h * (QT_KEYS / 4)), pk);
                        fa_wait_st();
                        fa_fence_before();
                        fa_arrive(fa_smem(h == 0 ? &p_half[t] : &p_full[t]));
                    }
                };
                if (__any_sync(0xffffffffu, apart)) weigh(std::true_type{});
                else weigh(std::false_type{});
                float l0, l1, l2, l3;
                fa_unpack2(l01, l0, l1);
                fa_unpack2(l23, l2, l3);
                l = fmaf((l0 + l1) + (l2 + l3), apart ? 1.0f : exp2f(r - values), l);
            }
            // ---- the item's result, or a part of it ----
            if (ok && part_of) {
                if (!wait(&o_done[t], items++)) break;
                fa_fence_after();
                const bool whole = at.off == 0 && at.part == at.n;
                const float up_r = exp2f(r), inv = l == 0.0f ? 0.0f : up_r / l;
                __nv_bfloat16* o = a.out + ((long long)(at.row.tok0 + qrow) * a.n_heads + at.head) * HD;
                // (the first slot if another block began the item, else the second)
                float* slot = a.slots + (2 * (size_t)blockIdx.x + (at.off > 0 ? 0 : 1)) * qt_slot_floats(HD);
                const int irow = t * QT_Q + trow;
#pragma unroll 1
                for (int c0 = 0; c0 < HD; c0 += 32) {
                    uint32_t w[32];
                    fa_ld32(o_addr + (uint32_t)c0, w);
                    fa_wait_ld();
                    if (whole && real) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint32_t v[4];
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(w[e + 2 * h]) * inv,
                                                                              __uint_as_float(w[e + 2 * h + 1]) * inv);
                                v[h] = *reinterpret_cast<const uint32_t*>(&x);
                            }
                            *reinterpret_cast<uint4*>(o + c0 + e) = make_uint4(v[0], v[1], v[2], v[3]);
                        }
                    } else if (!whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(slot + ((size_t)((c0 + e) >> 2) * QT_ITEM + irow) * 4) =
                                make_float4(__uint_as_float(w[e]) * up_r, __uint_as_float(w[e + 1]) * up_r,
                                            __uint_as_float(w[e + 2]) * up_r, __uint_as_float(w[e + 3]) * up_r);
                    }
                }
                if (!whole) {
                    slot[(size_t)QT_ITEM * HD + irow] = m;
                    slot[(size_t)QT_ITEM * (HD + 1) + irow] = l;
                }
                fa_fence_before();                       // (the next item's products may write O from here on)
            }
            if (!ok || !at.next(a)) break;
        }
    }
    __syncwarp();
    fa_fence_before();
    __syncthreads();
    if (*abort_flag && tid == 0) {
        atomicOr(a.status, MF_STATUS_WAIT_TIMEOUT);
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ------------------------------------------------------------------------------------------
// join: the items that several blocks have worked on, in the blocks' order.  Block (c, g) joins rows 32 g .. of the
// item that block c + 1 began in, if it was the second to work on it; a lane takes a row, a warp a part of
// its dimensions.
// ------------------------------------------------------------------------------------------
#define QJ_WARPS 8
template <int HD>
__global__ void __launch_bounds__(QJ_WARPS * 32) attention_q8_tc_join_kernel(QtArgs a) {
    pdl_launch_dependents();
    constexpr int EACH = HD / 4 / QJ_WARPS;               // groups of four dimensions a warp
    const int c = blockIdx.x + 1, warp = threadIdx.x >> 5, irow = blockIdx.y * 32 + (threadIdx.x & 31);
    pdl_wait();
    const int4 first = a.first[c];                        // row, item, tile, share
    if (first.w == 0 || first.z == 0 || first.z > first.w) return;
    const QtRow row = qt_row(a, first.x);
    const int group = first.y / a.n_heads, head = first.y - group * a.n_heads, qrow = group * QT_ITEM + irow;
    if (qrow >= row.count) return;
    int lo, n;
    qt_tiles(a, row, group * QT_ITEM, &lo, &n);
    const int c0 = c - 1, c1 = c + (n - first.z - 1) / first.w;
    float m = -INFINITY, l = 0.0f;
    float4 o[EACH];
#pragma unroll
    for (int e = 0; e < EACH; ++e) o[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int b = c0; b <= c1; ++b) {
        const float* slot = a.slots + (2 * (size_t)b + (b == c0 ? 1 : 0)) * qt_slot_floats(HD);
        const float ms = slot[(size_t)QT_ITEM * HD + irow], ls = slot[(size_t)QT_ITEM * (HD + 1) + irow];
        float4 x[EACH];
#pragma unroll
        for (int e = 0; e < EACH; ++e)
            x[e] = *reinterpret_cast<const float4*>(slot + ((size_t)(warp * EACH + e) * QT_ITEM + irow) * 4);
        const float top = fmaxf(m, ms), use = top == -INFINITY ? 0.0f : top;
        const float keep = exp2f(m - use), f = exp2f(ms - use);
        m = top;
        l = fmaf(ls, f, l * keep);
#pragma unroll
        for (int e = 0; e < EACH; ++e) {
            o[e].x = fmaf(x[e].x, f, o[e].x * keep); o[e].y = fmaf(x[e].y, f, o[e].y * keep);
            o[e].z = fmaf(x[e].z, f, o[e].z * keep); o[e].w = fmaf(x[e].w, f, o[e].w * keep);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    __nv_bfloat16* to = a.out + ((long long)(row.tok0 + qrow) * a.n_heads + head) * HD + warp * EACH * 4;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
        const __nv_bfloat162 x = __floats2bfloat162_rn(o[e].x * inv, o[e].y * inv);
        const __nv_bfloat162 y = __floats2bfloat162_rn(o[e].z * inv, o[e].w * inv);
        *reinterpret_cast<uint2*>(to + 4 * e) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
}

// ---- host side ------------------------------------------------------------------------------
static int qt_map(CUtensorMap* map, const void* ptr, long long rows, long long width) {
    FaEncodeFn fn = fa_encode_fn();
    if (!fn) return MF_ERR_NO_TENSORMAP;
    if (rows <= 0 || rows > 0x7fffffffLL) return MF_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)width * 2};
    cuuint32_t box[2] = {64, 128};
    cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : MF_ERR_TENSORMAP;
}

// The scratch's parts, one behind the other; returns its size in bytes.
static long long qt_layout(QtArgs* a, uint8_t* base, int n_tokens, int n_rows, int stretch, int n_heads, int n_kv, int hd) {
    long long at = 0;
    auto take = [&](long long bytes) {
        uint8_t* p = base + at;
        at += (bytes + 1023) & ~1023LL;
        return p;
    };
    const long long vectors = (long long)n_rows * n_kv * stretch, queries = (long long)n_tokens * n_heads;
    const int blocks = mf_sm_count();
    // (the queries first: calls over other rows of the step find them in the same place)
    a->q16 = (__half*)take(queries * hd * 2);
    a->factor = (float*)take(queries * 4);
    a->first = (int4*)take(blocks * 16LL);
    a->slots = (float*)take(2LL * blocks * (long long)qt_slot_floats(hd) * 4);
    a->k16 = (__half*)take(vectors * hd * 2);
    a->v16 = (__half*)take(vectors * hd * 2);
    a->powers = (float2*)take(vectors / QT_KEYS * 8);
    a->own = (float*)take(vectors * 8);
    return at;
}
// Bytes of scratch of a call over `n_rows` rows whose tokens see `stretch` positions (a multiple of 128).
extern "C" long long mf_attention_q8_tc_scratch(int n_tokens, int n_rows, int stretch, int n_heads, int n_kv, int hd) {
    QtArgs a{};
    return qt_layout(&a, nullptr, n_tokens, n_rows, stretch, n_heads, n_kv, hd);
}

template <int HD> static int qt_launch(const QtArgs& a, int fmt, cudaStream_t stream) {
    CUtensorMap mq, mk, mv;
    const long long vectors = (long long)a.n_rows * a.n_kv * a.stretch;
    if (int e = qt_map(&mq, a.q16, a.n_tokens, (long long)a.n_heads * HD)) return e;
    if (int e = qt_map(&mk, a.k16, vectors, HD)) return e;
    if (int e = qt_map(&mv, a.v16, vectors, HD)) return e;
    constexpr int used = (HD / 64) * 16384 * 6 + 1024 + 256;
    // (tensor memory is allocated whole: no other block with some may share the SM)
    constexpr int smem = used > MF_TMEM_SMEM_ALONE ? used : MF_TMEM_SMEM_ALONE;
    static bool opened[64] = {};
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    if (dev < 0 || dev >= 64 || !opened[dev]) {
        if (cudaError_t e = cudaFuncSetAttribute(attention_q8_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))
            return (int)e;
        if (dev >= 0 && dev < 64) opened[dev] = true;
    }
    const long long tiles = vectors / QT_KEYS * 2;
    const long long queries = a.with_q ? ((long long)a.n_tokens * a.n_heads + QU_VECTORS - 1) / QU_VECTORS : 0;
    if (tiles + queries > 0x7fffffffLL) return MF_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(tiles + queries));
    if (fmt == MF_Q8_E4M3) mf_launch(q8_unpack_kernel<MF_Q8_E4M3, HD>, grid, dim3(QU_THREADS), 0, stream, a, (int)tiles);
    else mf_launch(q8_unpack_kernel<MF_Q8_INT8, HD>, grid, dim3(QU_THREADS), 0, stream, a, (int)tiles);
    if (int e = MF_LAUNCH_CHECK()) return e;
    const int blocks = mf_sm_count();
    mf_launch(attention_q8_tc_kernel<HD>, dim3(blocks), dim3(QT_THREADS), smem, stream, mq, mk, mv, a);
    if (int e = MF_LAUNCH_CHECK()) return e;
    if (blocks > 1) mf_launch(attention_q8_tc_join_kernel<HD>, dim3(blocks - 1, QT_ITEM / 32), dim3(QJ_WARPS * 32), 0, stream, a);
    return MF_LAUNCH_CHECK();
}

// `scratch`: what mf_attention_q8_tc_scratch says, 1024-byte aligned.  `with_q` 0: the scratch holds the queries of
// these tokens already, from a call over other rows of the step.
extern "C" int mf_attention_q8_tc(const void* q, const void* k_codes, const void* v_codes, const float* k_scales,
                                  const float* v_scales, const int* cu_seqlens, const int* seq_end, const int* page_table,
                                  int table_stride, int ring, int n_pages, void* out, void* scratch, int n_tokens, int n_rows,
                                  int max_end, int stretch, int n_heads, int n_kv, int hd, int window, float scale, int fmt,
                                  int with_q, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0 || n_rows <= 0) return 0;
    if ((hd != 64 && hd != 128) || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0) return MF_ERR_UNSUPPORTED;
    if (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8) return MF_ERR_UNSUPPORTED;
    if (table_stride <= 0 || n_pages <= 0 || ring < 0 || ring % MF_PAGE != 0 || window < 0 || (ring > 0 && window <= 0) ||
        status == nullptr || stretch <= 0 || stretch % QT_KEYS != 0 || max_end <= 0)
        return MF_ERR_ARGUMENT;
    if (table_stride > (1 << 24) || max_end > (1 << 30)) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_codes | (uintptr_t)v_codes) & 15) return MF_ERR_UNSUPPORTED;
    if (scratch == nullptr || ((uintptr_t)scratch & 1023)) return MF_ERR_ARGUMENT;
    // (tiles of all items are counted in 32 bits)
    if (((long long)n_tokens / QT_ITEM + n_rows) * n_heads * (stretch / QT_KEYS) > 0x7fffffffLL ||
        (long long)n_rows * n_kv * stretch > 0x7fffffffLL)
        return MF_ERR_UNSUPPORTED;
    QtArgs a{};
    a.q = (const __nv_bfloat16*)q; a.k_codes = (const uint8_t*)k_codes; a.v_codes = (const uint8_t*)v_codes;
    a.k_scales = k_scales; a.v_scales = v_scales; a.cu_seqlens = cu_seqlens; a.seq_end = seq_end;
    a.page_table = page_table; a.table_stride = table_stride; a.ring = ring; a.n_pages = n_pages;
    a.max_end = ring > 0 || max_end < table_stride * MF_PAGE ? max_end : table_stride * MF_PAGE;
    a.stretch = stretch; a.out = (__nv_bfloat16*)out; a.n_tokens = n_tokens; a.n_rows = n_rows; a.n_heads = n_heads;
    a.n_kv = n_kv; a.window = window; a.with_q = with_q; a.scale = scale; a.status = status;
    qt_layout(&a, (uint8_t*)scratch, n_tokens, n_rows, stretch, n_heads, n_kv, hd);
    return hd == 64 ? qt_launch<64>(a, fmt, stream) : qt_launch<128>(a, fmt, stream);
}
