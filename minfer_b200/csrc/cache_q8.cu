// Keys and values in 8 bits: written into pages as they come off the projection, and read back.
// (q8.cuh says what a vector's codes and scale are.)
//
// Storage of a cache entry: codes [page][kv_head][64][hd] for K and for V, one byte each, and
// scales [page][kv_head][64] in float32.
#include "q8.cuh"

// ------------------------------------------------------------------------------------------
// Rotary on q and k, then k and v quantised and written to the pages (the pairs, the angles and the
// sums over a projection's K splits are those of rope_kvstore in ops.cu).
//
// The float32 values of a vector stay in registers between the reduction to its largest magnitude and the
// rounding, so a code is rounded once, from float32, whatever type the activations have.  Magnitudes are
// compared as integers (the order of non-negative floats), which keeps NaN above infinity above
// everything finite; fmaxf would drop it.  Bound by bytes for prompts and by latency for single tokens.
//
// Two kernels: pairs (i, i + hd/2) of fully rotated heads of 64, 128 or 256 in wide accesses
// (rope_kvstore_q8_wide_kernel), and any even hd up to 256, any rotated part, either pairing.
// ------------------------------------------------------------------------------------------
struct StoreQ8Args {
    const float* qkv;              // [n_partials or 1][tokens][(n_heads + 2 n_kv) * hd]
    int n_partials, n_tokens;
    const float* bias;
    const int* positions;
    const int* token_row;
    const int* seq_end;
    const double* inv_freq;
    void* q_out;                   // [tokens][n_heads][hd]
    void* k_out;                   // [tokens][n_kv][hd] or null
    void* v_out;
    uint8_t* k_codes;
    uint8_t* v_codes;
    float* k_scales;
    float* v_scales;
    const int* page_table;
    int table_stride, ring, n_pages;
    int n_heads, n_kv, hd, rotary_dim, style;
    unsigned* status;
};

// Where a token's keys and values go: the place [page][0][pos % 64] in vectors, -1 if they are not kept (a ring
// keeps a sequence's last positions) or have no page, which sets the status bit.
__device__ __forceinline__ long long q8_place(const StoreQ8Args& a, int t, int pos, bool tell) {
    const int b = a.token_row[t];
    if (a.ring > 0 && pos < a.seq_end[b] - a.ring) return -1;
    const int index = (a.ring > 0 ? pos % a.ring : pos) >> 6;
    const int page = pos >= 0 && index < a.table_stride ? a.page_table[(size_t)b * a.table_stride + index] : -1;
    if (page < 0 || page >= a.n_pages) {
        if (tell) atomicOr(a.status, MF_STATUS_BAD_POSITION);
        return -1;
    }
    return (long long)page * a.n_kv * MF_PAGE + (pos & (MF_PAGE - 1));
}
__device__ __forceinline__ float2 q8_turn(int pos, double inv_freq) {        // (cos, sin)
    const double two_pi = 6.283185307179586476925286766559;
    const double th = (double)pos * inv_freq;
    float sn, cs;
    sincosf((float)(th - two_pi * floor(th / two_pi)), &sn, &cs);
    return make_float2(cs, sn);
}
// scale and the factor of a vector whose largest magnitude has the bits `top`
template <int FMT> __device__ __forceinline__ float q8_scale(unsigned top, float* by) {
    if (top >= 0x7f800000u) {
        *by = 0.0f;
        return __uint_as_float(0x7fc00000u);
    }
    const float big = fmaxf(__uint_as_float(top), MF_Q8_TINY);
    *by = q8_limit<FMT>() / big;
    return big / q8_limit<FMT>();
}
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ void add4(float4& x, const float4& y) { x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w; }
template <typename T> __device__ __forceinline__ void store4(T* p, const float* v);
template <> __device__ __forceinline__ void store4<float>(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <> __device__ __forceinline__ void store4<__nv_bfloat16>(__nv_bfloat16* p, const float* v) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(v[0], v[1]), y = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// A lane takes four neighbouring pairs, hd / 8 lanes a vector; a block takes `tokens` tokens, whose sines
// and cosines it forms once for all heads (a thread each where a block has enough tokens), or a part of one
// token's heads (blockIdx.y) where tokens are few.  2,048 tokens of 28 heads and 4 of 128, written and their
// 128 pages a head read back in a second launch: 18.4 us for 65 MB; with registers for 6 blocks an SM 24.6.
// SPLIT: the projection left K splits, whose sums keep every load of a thread in flight at once; without them
// few registers, so that many blocks share an SM.
template <typename T, int FMT, int HD, bool SPLIT>
__global__ void __launch_bounds__(128, SPLIT ? 6 : 16) rope_kvstore_q8_wide_kernel(StoreQ8Args a, int tokens) {
    // the step's integers and weights are read before the wait, the projection behind it
    pdl_launch_dependents();
    constexpr int LPH = HD / 8, GROUPS = 128 / LPH, HALF = HD / 2, MOST = 128 / HALF;
    __shared__ float2 cs_s[128];               // [token][HALF]
    __shared__ long long place_s[MOST];
    const int t0 = blockIdx.x * tokens, here = min(tokens, a.n_tokens - t0), tid = threadIdx.x;
    for (int i = tid; i < here * HALF; i += 128) cs_s[i] = q8_turn(a.positions[t0 + i / HALF], a.inv_freq[i % HALF]);
    if (tid < here) place_s[tid] = q8_place(a, t0 + tid, a.positions[t0 + tid], blockIdx.y == 0);
    __syncthreads();
    pdl_wait();
    const int n_all = a.n_heads + 2 * a.n_kv, l = tid % LPH;
    const size_t plane = (size_t)a.n_tokens * n_all * HD;
    const float* in = a.qkv + (size_t)t0 * n_all * HD + 4 * l;
    for (int u = blockIdx.y * GROUPS + tid / LPH; u < here * n_all; u += gridDim.y * GROUPS) {
        const int k = u / n_all, head = u - k * n_all;
        const float* p = in + (size_t)u * HD;
        float4 x = *reinterpret_cast<const float4*>(p), y = *reinterpret_cast<const float4*>(p + HALF);
        // splits in split order, four of them asked for at a time
        for (int s0 = 1; SPLIT && s0 < a.n_partials; s0 += 4) {
            float4 px[4], py[4];
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (s0 + s < a.n_partials) {
                    px[s] = *reinterpret_cast<const float4*>(p + (s0 + s) * plane);
                    py[s] = *reinterpret_cast<const float4*>(p + (s0 + s) * plane + HALF);
                }
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (s0 + s < a.n_partials) { add4(x, px[s]); add4(y, py[s]); }
        }
        if (a.bias != nullptr) {
            add4(x, *reinterpret_cast<const float4*>(a.bias + head * HD + 4 * l));
            add4(y, *reinterpret_cast<const float4*>(a.bias + head * HD + HALF + 4 * l));
        }
        float lo[4] = {x.x, x.y, x.z, x.w}, hi[4] = {y.x, y.y, y.z, y.w};
        const bool is_v = head >= a.n_heads + a.n_kv, is_q = head < a.n_heads;
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 cs = cs_s[k * HALF + 4 * l + j];
                const float c = lo[j], d = hi[j];
                lo[j] = c * cs.x - d * cs.y;
                hi[j] = c * cs.y + d * cs.x;
            }
        }
        T* dense = nullptr;                    // the activations' type: q, or the step's own k and v
        const int hk = is_v ? head - a.n_heads - a.n_kv : head - a.n_heads;
        if (is_q) dense = (T*)a.q_out + ((size_t)(t0 + k) * a.n_heads + head) * HD;
        else if (void* step = is_v ? a.v_out : a.k_out) dense = (T*)step + ((size_t)(t0 + k) * a.n_kv + hk) * HD;
        if (dense != nullptr) {
            store4<T>(dense + 4 * l, lo);
            store4<T>(dense + HALF + 4 * l, hi);
        }
        // (lanes of one vector take the same way; the reduction names them alone)
        if (is_q || place_s[k] < 0) continue;
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, max(magnitude(lo[j]), magnitude(hi[j])));
        const unsigned group = (LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1u) << (tid & 31 & ~(LPH - 1)));
        top = __reduce_max_sync(group, top);
        float by;
        const float scale = q8_scale<FMT>(top, &by);
        const long long at = place_s[k] + (long long)hk * MF_PAGE;
        uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + at * HD + 4 * l;
        if (l == 0) (is_v ? a.v_scales : a.k_scales)[at] = scale;
        if (by == 0.0f) {
#pragma unroll
            for (int j = 0; j < 4; ++j) lo[j] = hi[j] = 0.0f;
        }
        *reinterpret_cast<uint32_t*>(codes) = q8_pack2<FMT>(lo[0] * by, lo[1] * by) | q8_pack2<FMT>(lo[2] * by, lo[3] * by) << 16;
        *reinterpret_cast<uint32_t*>(codes + HALF) = q8_pack2<FMT>(hi[0] * by, hi[1] * by) | q8_pack2<FMT>(hi[2] * by, hi[3] * by) << 16;
    }
}

// A warp takes a head of a token, a lane the pairs lane, lane + 32, ...
template <typename T, int FMT>
__global__ void __launch_bounds__(128) rope_kvstore_q8_kernel(StoreQ8Args a) {
    pdl_launch_dependents();
    __shared__ float2 cs_s[128];
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = a.positions[t], half = a.hd >> 1;
    const int rhalf = a.inv_freq != nullptr ? a.rotary_dim >> 1 : 0;
    for (int i = threadIdx.x; i < rhalf; i += blockDim.x) cs_s[i] = q8_turn(pos, a.inv_freq[i]);
    const long long place = q8_place(a, t, pos, threadIdx.x == 0 && blockIdx.y == 0);
    __syncthreads();
    pdl_wait();
    const int n_all = a.n_heads + 2 * a.n_kv;
    const size_t width = (size_t)n_all * a.hd, plane = (size_t)a.n_tokens * width;
    for (int head = blockIdx.y * 4 + warp; head < n_all; head += gridDim.y * 4) {
        const bool is_v = head >= a.n_heads + a.n_kv;
        const float* in = a.qkv + (size_t)t * width + (size_t)head * a.hd;
        const int hk = is_v ? head - a.n_heads - a.n_kv : head - a.n_heads;
        T* dense = nullptr;
        if (head < a.n_heads) dense = (T*)a.q_out + ((size_t)t * a.n_heads + head) * a.hd;
        else if (void* step = is_v ? a.v_out : a.k_out) dense = (T*)step + ((size_t)t * a.n_kv + hk) * a.hd;
        float v[4][2];
        int d[4][2];
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = lane + 32 * j;
            v[j][0] = v[j][1] = 0.0f;
            if (i >= half) continue;
            const bool turned = !is_v && i < rhalf;
            d[j][0] = turned ? (a.style == 0 ? i : 2 * i) : is_v ? 2 * i : 2 * rhalf + 2 * (i - rhalf);
            d[j][1] = turned && a.style == 0 ? i + rhalf : d[j][0] + 1;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = in[d[j][e]];
                for (int s = 1; s < a.n_partials; ++s) x += in[s * plane + d[j][e]];
                if (a.bias != nullptr) x += a.bias[head * a.hd + d[j][e]];
                v[j][e] = x;
            }
            if (turned) {
                const float2 cs = cs_s[i];
                const float x = v[j][0], y = v[j][1];
                v[j][0] = x * cs.x - y * cs.y;
                v[j][1] = x * cs.y + y * cs.x;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (dense != nullptr) dense[d[j][e]] = from_f32<T>(v[j][e]);
                top = max(top, magnitude(v[j][e]));
            }
        }
        if (head < a.n_heads || place < 0) continue;           // uniform over the warp
        top = __reduce_max_sync(0xffffffffu, top);
        float by;
        const float scale = q8_scale<FMT>(top, &by);
        const long long at = place + (long long)hk * MF_PAGE;
        uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + at * a.hd;
        if (lane == 0) (is_v ? a.v_scales : a.k_scales)[at] = scale;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (lane + 32 * j >= half) continue;
            const uint32_t c = by == 0.0f ? 0u : q8_pack2<FMT>(v[j][0] * by, v[j][1] * by);
            codes[d[j][0]] = (uint8_t)c;
            codes[d[j][1]] = (uint8_t)(c >> 8);
        }
    }
}

template <typename T, int FMT, int HD> static int store_wide(const StoreQ8Args& a, cudaStream_t stream) {
    constexpr int groups = 128 / (HD / 8), most = 128 / (HD / 2);
    const int n_all = a.n_heads + 2 * a.n_kv, fill = 4 * mf_sm_count();
    // as many tokens a block as its threads form sines for, unless the GPU is not full then
    int tokens = most;
    while (tokens > 1 && a.n_tokens / tokens < fill) tokens >>= 1;
    const int blocks = (a.n_tokens + tokens - 1) / tokens;
    int gy = blocks >= fill ? 1 : (fill + blocks - 1) / blocks;
    if (gy > (tokens * n_all + groups - 1) / groups) gy = (tokens * n_all + groups - 1) / groups;
    if (a.n_partials > 1)
        mf_launch(rope_kvstore_q8_wide_kernel<T, FMT, HD, true>, dim3(blocks, gy), dim3(128), 0, stream, a, tokens);
    else
        mf_launch(rope_kvstore_q8_wide_kernel<T, FMT, HD, false>, dim3(blocks, gy), dim3(128), 0, stream, a, tokens);
    return MF_LAUNCH_CHECK();
}
template <typename T, int FMT> static int store_launch(const StoreQ8Args& a, bool wide, cudaStream_t stream) {
    if (wide)
        return a.hd == 64 ? store_wide<T, FMT, 64>(a, stream) : a.hd == 128 ? store_wide<T, FMT, 128>(a, stream)
                                                                            : store_wide<T, FMT, 256>(a, stream);
    const int n_all = a.n_heads + 2 * a.n_kv;
    int gy = (4 * mf_sm_count() + a.n_tokens - 1) / a.n_tokens;
    if (gy > (n_all + 3) / 4) gy = (n_all + 3) / 4;
    mf_launch(rope_kvstore_q8_kernel<T, FMT>, dim3(a.n_tokens, gy), dim3(128), 0, stream, a);
    return MF_LAUNCH_CHECK();
}

extern "C" int mf_rope_kvstore_q8(const float* qkv, int n_partials, const float* bias, const int* positions,
                                  const int* token_row, const int* seq_end, const double* inv_freq, void* q_out,
                                  void* k_out, void* v_out, void* k_codes, void* v_codes, float* k_scales,
                                  float* v_scales, const int* page_table, int table_stride, int ring, int n_pages,
                                  int n_tokens, int n_heads, int n_kv, int hd, int rotary_dim, int style, int dtype,
                                  int fmt, unsigned* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (hd % 2 != 0 || hd < 2 || hd > 256 || rotary_dim % 2 != 0 || rotary_dim > hd || rotary_dim < 0 ||
        n_heads < 0 || n_kv <= 0)
        return MF_ERR_UNSUPPORTED;
    if (ring < 0 || ring % MF_PAGE != 0 || table_stride <= 0 || n_pages <= 0 || (style != 0 && style != 1))
        return MF_ERR_ARGUMENT;
    if ((dtype != MF_DTYPE_F32 && dtype != MF_DTYPE_BF16) || (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8))
        return MF_ERR_UNSUPPORTED;
    StoreQ8Args a{};
    a.qkv = qkv; a.n_partials = n_partials; a.n_tokens = n_tokens; a.bias = bias; a.positions = positions;
    a.token_row = token_row; a.seq_end = seq_end; a.inv_freq = inv_freq; a.q_out = q_out; a.k_out = k_out;
    a.v_out = v_out; a.k_codes = (uint8_t*)k_codes; a.v_codes = (uint8_t*)v_codes; a.k_scales = k_scales;
    a.v_scales = v_scales; a.page_table = page_table; a.table_stride = table_stride; a.ring = ring;
    a.n_pages = n_pages; a.n_heads = n_heads; a.n_kv = n_kv; a.hd = hd; a.rotary_dim = rotary_dim; a.style = style;
    a.status = status;
    // wide accesses need their addresses aligned (rows are multiples of 64 elements)
    const uintptr_t bits = (uintptr_t)qkv | (uintptr_t)bias | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out;
    const bool wide = inv_freq != nullptr && style == 0 && rotary_dim == hd && (hd == 64 || hd == 128 || hd == 256) &&
                      (bits & 15) == 0 && (((uintptr_t)k_codes | (uintptr_t)v_codes) & 3) == 0;
    if (dtype == MF_DTYPE_F32)
        return fmt == MF_Q8_E4M3 ? store_launch<float, MF_Q8_E4M3>(a, wide, stream)
                                 : store_launch<float, MF_Q8_INT8>(a, wide, stream);
    return fmt == MF_Q8_E4M3 ? store_launch<__nv_bfloat16, MF_Q8_E4M3>(a, wide, stream)
                             : store_launch<__nv_bfloat16, MF_Q8_INT8>(a, wide, stream);
}

// ------------------------------------------------------------------------------------------
// Pages read back: out [rows * table_stride][n_kv][64][hd] in bfloat16 or float32, a row's pages in the order
// of the page table; places that hold no position of the row are zeros.
//
// Bound by bytes: 1 read and 2 (4) written an element.  A block takes one page of one key/value
// head, K or V: a thread's unit is 8 codes, so that a warp's stores are whole lines without gaps (16 codes,
// two stores a thread: 72 us where this takes 62), and all of a thread's loads of a round are
// issued before the first conversion.  4 sequences of 15,001 to 31,999 positions, 4 heads of 128, in a table
// of 500 pages a row: 62.5 us = 5.8 TB/s of what is read and written, the zeros behind the shorter rows included.
// ------------------------------------------------------------------------------------------
struct ReadQ8Args {
    const uint8_t* k_codes;
    const uint8_t* v_codes;
    const float* k_scales;
    const float* v_scales;
    const int* page_table;
    int table_stride, ring, n_pages;
    const int* seq_end;
    void* k_out;
    void* v_out;
    int rows, n_kv, hd;
    int fill;                      // 1: pages that hold nothing of their row are written as zeros too
    unsigned* status;
};

#define RD_THREADS 256
template <typename T> __device__ __forceinline__ void store8(T* p, const float* v);
template <> __device__ __forceinline__ void store8<float>(float* p, const float* v) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T, int FMT>
__global__ void __launch_bounds__(RD_THREADS) read_pages_q8_kernel(ReadQ8Args a) {
    pdl_launch_dependents();
    const int hk = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int row = blockIdx.x / a.table_stride, index = blockIdx.x - row * a.table_stride;
    const int end = a.seq_end[row];
    const int page = a.page_table[blockIdx.x];
    // places [0, n) of the page hold positions of the row (a ring that is full: all of them; the ring's
    // lap does not matter to what a place holds)
    const int span = min(a.ring > 0 ? min(end, a.ring) : end, a.table_stride * MF_PAGE);
    int n = min(MF_PAGE, span - index * MF_PAGE);
    // (a length beyond the table)
    if (a.ring == 0 && end > span && index == 0 && hk == 0 && threadIdx.x == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
    if (n <= 0 && !a.fill) { pdl_wait(); return; }
    const bool there = page >= 0 && page < a.n_pages;
    if (n > 0 && !there) {
        if (threadIdx.x == 0 && hk == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
        n = 0;
    }
    pdl_wait();
    const int upr = a.hd >> 3;                        // units of 8 codes a vector
    const int units = MF_PAGE * upr;
    const long long from = there ? ((long long)page * a.n_kv + hk) * MF_PAGE : 0;
    const uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + from * a.hd;
    const float* scales = (is_v ? a.v_scales : a.k_scales) + from;
    T* out = (T*)(is_v ? a.v_out : a.k_out) + ((long long)blockIdx.x * a.n_kv + hk) * MF_PAGE * a.hd;
    for (int u0 = threadIdx.x; u0 < units; u0 += 4 * RD_THREADS) {
        uint2 w[4];
        float s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = u0 + i * RD_THREADS, place = u / upr;
            w[i] = make_uint2(0, 0);
            s[i] = 0.0f;
            if (u < units && place < n) {
                w[i] = *reinterpret_cast<const uint2*>(codes + (long long)u * 8);
                s[i] = scales[place];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int u = u0 + i * RD_THREADS;
            if (u >= units) continue;
            const uint32_t words[2] = {w[i].x, w[i].y};
            float v[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) q8_floats<FMT>(words[j], v + 4 * j);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= s[i];
            store8<T>(out + (long long)u * 8, v);
        }
    }
}

template <typename T, int FMT> static int read_launch(const ReadQ8Args& a, cudaStream_t stream) {
    const dim3 grid((unsigned)(a.rows * a.table_stride), a.n_kv, 2);
    mf_launch(read_pages_q8_kernel<T, FMT>, grid, dim3(RD_THREADS), 0, stream, a);
    return MF_LAUNCH_CHECK();
}

extern "C" int mf_read_pages_q8(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales,
                                const int* page_table, int table_stride, int ring, int n_pages,
                                const int* seq_end, void* k_out, void* v_out, int rows, int n_kv, int hd, int dtype,
                                int fmt, int fill, unsigned* status, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (hd % 16 != 0 || hd < 16 || hd > 256 || n_kv <= 0 || n_kv > 65535) return MF_ERR_UNSUPPORTED;
    if (ring < 0 || ring % MF_PAGE != 0 || table_stride <= 0 || n_pages <= 0)
        return MF_ERR_ARGUMENT;
    if ((long long)rows * table_stride > 0x7fffffffLL || table_stride > 0x7fffffff / MF_PAGE) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return MF_ERR_UNSUPPORTED;
    if ((dtype != MF_DTYPE_F32 && dtype != MF_DTYPE_BF16) || (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8))
        return MF_ERR_UNSUPPORTED;
    ReadQ8Args a{};
    a.k_codes = (const uint8_t*)k_codes; a.v_codes = (const uint8_t*)v_codes; a.k_scales = k_scales;
    a.v_scales = v_scales; a.page_table = page_table; a.table_stride = table_stride;
    a.ring = ring; a.n_pages = n_pages; a.seq_end = seq_end; a.k_out = k_out; a.v_out = v_out; a.rows = rows;
    a.n_kv = n_kv; a.hd = hd; a.fill = fill; a.status = status;
    if (dtype == MF_DTYPE_F32)
        return fmt == MF_Q8_E4M3 ? read_launch<float, MF_Q8_E4M3>(a, stream)
                                 : read_launch<float, MF_Q8_INT8>(a, stream);
    return fmt == MF_Q8_E4M3 ? read_launch<__nv_bfloat16, MF_Q8_E4M3>(a, stream)
                             : read_launch<__nv_bfloat16, MF_Q8_INT8>(a, stream);
}
