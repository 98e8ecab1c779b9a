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
// A warp owns one head of one token: a vector's largest magnitude is then one warp reduction, and
// the float32 values stay in registers between it and the rounding, so a code is rounded once, from
// float32, whatever type the activations have.  Magnitudes are compared as integers (the order of
// non-negative floats), which keeps NaN above infinity above everything finite; fmaxf would drop it.
//
// VP > 0: pairs (i, i + hd/2) of a fully rotated head, hd = 64 VP, a lane takes VP neighbouring ones,
// so that loads are 4 VP and stores 2 VP bytes a lane without gaps in the warp; VP = 0: any even
// hd up to 256, any rotated part, either pairing, a lane takes pairs lane, lane + 32, ...
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

template <typename T, int N> __device__ __forceinline__ void store_n(T* p, const float* v) {
    if (N == 1) { p[0] = from_f32<T>(v[0]); return; }
    if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            *reinterpret_cast<float2*>(reinterpret_cast<float*>(p) + i) = make_float2(v[i], v[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2)
            *reinterpret_cast<__nv_bfloat162*>(reinterpret_cast<__nv_bfloat16*>(p) + i) =
                __floats2bfloat162_rn(v[i], v[i + 1]);
    }
}
template <int N> __device__ __forceinline__ void load_n(const float* p, float* v) {
    if (N == 1) v[0] = p[0];
    if (N == 2) { const float2 x = *reinterpret_cast<const float2*>(p); v[0] = x.x; v[1] = x.y; }
    if (N == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
}

template <typename T, int FMT, int VP>
__global__ void __launch_bounds__(128) rope_kvstore_q8_kernel(StoreQ8Args a) {
    // the step's integers and weights are read before the wait, the projection behind it
    pdl_launch_dependents();
    __shared__ float2 cs_table[128];
    const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pos = a.positions[t];
    const int hd = VP > 0 ? 64 * VP : a.hd, half = hd >> 1;
    const int rhalf = a.inv_freq != nullptr ? a.rotary_dim >> 1 : 0;
    for (int i = threadIdx.x; i < rhalf; i += blockDim.x) {
        const double two_pi = 6.283185307179586476925286766559;
        const double th = (double)pos * a.inv_freq[i];
        float sn, cs;
        sincosf((float)(th - two_pi * floor(th / two_pi)), &sn, &cs);
        cs_table[i] = make_float2(cs, sn);
    }
    long long slot = -1;                       // [page][0][pos % 64] in vectors, or -1: not kept
    {
        const int b = a.token_row[t];
        const bool keep = a.ring == 0 || pos >= a.seq_end[b] - a.ring;
        if (keep) {
            const int index = (a.ring > 0 ? pos % a.ring : pos) >> 6;
            const int page = pos >= 0 && index < a.table_stride ? a.page_table[(size_t)b * a.table_stride + index] : -1;
            if (page < 0 || page >= a.n_pages) {
                if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.status, MF_STATUS_BAD_POSITION);
            } else {
                slot = (long long)page * a.n_kv * MF_PAGE + (pos & (MF_PAGE - 1));
            }
        }
    }
    __syncthreads();
    pdl_wait();
    const int n_all = a.n_heads + 2 * a.n_kv;
    const size_t width = (size_t)n_all * hd, plane = (size_t)a.n_tokens * width;
    const float* in = a.qkv + (size_t)t * width;
    constexpr int NP = VP > 0 ? VP : 4;        // pairs a lane holds
    constexpr int N = VP > 0 ? VP : 1;         // of them neighbours
    for (int head = blockIdx.y * 4 + warp; head < n_all; head += gridDim.y * 4) {
        const bool is_v = head >= a.n_heads + a.n_kv;
        float lo[NP], hi[NP];
        int d0[NP / N], d1[NP / N];            // where each run of neighbours begins
#pragma unroll
        for (int j = 0; j < NP / N; ++j) {
            const int i = VP > 0 ? lane * VP : lane + 32 * j;
            if (VP > 0) {
                d0[j] = i; d1[j] = i + half;
            } else if (i >= half) {
                d0[j] = d1[j] = -1;
            } else if (!is_v && i < rhalf) {
                d0[j] = a.style == 0 ? i : 2 * i;
                d1[j] = a.style == 0 ? i + rhalf : 2 * i + 1;
            } else {
                d0[j] = is_v ? 2 * i : 2 * rhalf + 2 * (i - rhalf);
                d1[j] = d0[j] + 1;
            }
        }
#pragma unroll
        for (int j = 0; j < NP / N; ++j) {
            if (d0[j] < 0) { lo[j] = hi[j] = 0.0f; continue; }
            const float* p = in + (size_t)head * hd;
            load_n<N>(p + d0[j], lo + j * N);
            load_n<N>(p + d1[j], hi + j * N);
        }
        // splits in split order, four of them asked for at a time
        for (int s0 = 1; s0 < a.n_partials; s0 += 4) {
            float pl[4][NP], ph[4][NP];
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int j = 0; j < NP / N; ++j)
                    if (s0 + s < a.n_partials && d0[j] >= 0) {
                        const float* p = in + (s0 + s) * plane + (size_t)head * hd;
                        load_n<N>(p + d0[j], pl[s] + j * N);
                        load_n<N>(p + d1[j], ph[s] + j * N);
                    }
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (s0 + s < a.n_partials)
#pragma unroll
                    for (int j = 0; j < NP; ++j)
                        if (d0[j / N] >= 0) { lo[j] += pl[s][j]; hi[j] += ph[s][j]; }
        }
        if (a.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < NP / N; ++j)
                if (d0[j] >= 0) {
                    float bl[N], bh[N];
                    load_n<N>(a.bias + (size_t)head * hd + d0[j], bl);
                    load_n<N>(a.bias + (size_t)head * hd + d1[j], bh);
#pragma unroll
                    for (int e = 0; e < N; ++e) { lo[j * N + e] += bl[e]; hi[j * N + e] += bh[e]; }
                }
        }
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int i = VP > 0 ? lane * VP + j : lane + 32 * j;
                if (i < rhalf) {
                    const float cs = cs_table[i].x, sn = cs_table[i].y, x = lo[j], y = hi[j];
                    lo[j] = x * cs - y * sn;
                    hi[j] = x * sn + y * cs;
                }
            }
        }
        T* dense = nullptr;                    // the activations' type: q, or the step's own k and v
        const int hk = is_v ? head - a.n_heads - a.n_kv : head - a.n_heads;
        if (head < a.n_heads) dense = (T*)a.q_out + ((size_t)t * a.n_heads + head) * hd;
        else if (void* step = is_v ? a.v_out : a.k_out) dense = (T*)step + ((size_t)t * a.n_kv + hk) * hd;
        if (dense != nullptr) {
#pragma unroll
            for (int j = 0; j < NP / N; ++j)
                if (d0[j] >= 0) {
                    store_n<T, N>(dense + d0[j], lo + j * N);
                    store_n<T, N>(dense + d1[j], hi + j * N);
                }
        }
        if (head < a.n_heads || slot < 0) continue;        // uniform over the warp
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            top = max(top, __float_as_uint(lo[j]) & 0x7fffffffu);
            top = max(top, __float_as_uint(hi[j]) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        const bool bad = top >= 0x7f800000u;
        const float big = bad ? 1.0f : fmaxf(__uint_as_float(top), MF_Q8_TINY);
        const float inv = q8_limit<FMT>() / big;
        const long long at = slot + (long long)hk * MF_PAGE;
        uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + at * hd;
        if (lane == 0) (is_v ? a.v_scales : a.k_scales)[at] = bad ? __uint_as_float(0x7fc00000u) : big / q8_limit<FMT>();
#pragma unroll
        for (int j = 0; j < NP; ++j) { lo[j] = bad ? 0.0f : lo[j] * inv; hi[j] = bad ? 0.0f : hi[j] * inv; }
        if constexpr (N >= 2) {
            uint32_t cl[NP / 2], ch[NP / 2];
#pragma unroll
            for (int j = 0; j < NP / 2; ++j) {
                cl[j] = q8_pack2<FMT>(lo[2 * j], lo[2 * j + 1]);
                ch[j] = q8_pack2<FMT>(hi[2 * j], hi[2 * j + 1]);
            }
            if (N == 2) {
                *reinterpret_cast<uint16_t*>(codes + d0[0]) = (uint16_t)cl[0];
                *reinterpret_cast<uint16_t*>(codes + d1[0]) = (uint16_t)ch[0];
            } else {
                *reinterpret_cast<uint32_t*>(codes + d0[0]) = cl[0] | cl[NP / 2 - 1] << 16;
                *reinterpret_cast<uint32_t*>(codes + d1[0]) = ch[0] | ch[NP / 2 - 1] << 16;
            }
        } else {
#pragma unroll
            for (int j = 0; j < NP; ++j)
                if (d0[j] >= 0) {
                    const uint32_t c = q8_pack2<FMT>(lo[j], hi[j]);
                    codes[d0[j]] = (uint8_t)c;
                    codes[d1[j]] = (uint8_t)(c >> 8);
                }
        }
    }
}

template <typename T, int FMT>
static int store_launch(const StoreQ8Args& a, int vp, dim3 grid, cudaStream_t stream) {
    if (vp == 1) mf_launch(rope_kvstore_q8_kernel<T, FMT, 1>, grid, dim3(128), 0, stream, a);
    else if (vp == 2) mf_launch(rope_kvstore_q8_kernel<T, FMT, 2>, grid, dim3(128), 0, stream, a);
    else if (vp == 4) mf_launch(rope_kvstore_q8_kernel<T, FMT, 4>, grid, dim3(128), 0, stream, a);
    else mf_launch(rope_kvstore_q8_kernel<T, FMT, 0>, grid, dim3(128), 0, stream, a);
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
    const int n_all = n_heads + 2 * n_kv;
    // blocks enough to fill the GPU, each warp with one head of a few tokens and several of many
    int gy = (4 * mf_sm_count() + n_tokens - 1) / n_tokens;
    if (gy > (n_all + 3) / 4) gy = (n_all + 3) / 4;
    if (gy < 1) gy = 1;
    // neighbouring pairs in wide accesses need addresses to match (rows are multiples of 64 elements)
    const uintptr_t bits = (uintptr_t)qkv | (uintptr_t)bias | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)v_out;
    const bool wide = inv_freq != nullptr && style == 0 && rotary_dim == hd && (hd == 64 || hd == 128 || hd == 256) &&
                      (bits & 15) == 0 && (((uintptr_t)k_codes | (uintptr_t)v_codes) & 3) == 0;
    const int vp = wide ? hd / 64 : 0;
    const dim3 grid(n_tokens, gy);
    if (dtype == MF_DTYPE_F32)
        return fmt == MF_Q8_E4M3 ? store_launch<float, MF_Q8_E4M3>(a, vp, grid, stream)
                                 : store_launch<float, MF_Q8_INT8>(a, vp, grid, stream);
    return fmt == MF_Q8_E4M3 ? store_launch<__nv_bfloat16, MF_Q8_E4M3>(a, vp, grid, stream)
                             : store_launch<__nv_bfloat16, MF_Q8_INT8>(a, vp, grid, stream);
}

// ------------------------------------------------------------------------------------------
// Pages read back: out [rows * out_stride][n_kv][64][hd] in bfloat16 or float32, a row's pages in the order
// of the page table; places that hold no position of the row are zeros, and so are pages behind the
// table's.
//
// Bound by bytes: 1 read and 2 (4) written an element.  A block takes one page of one key/value
// head, K or V: a thread's unit is 16 codes (one 16-byte load), and all of a thread's loads of a
// round are issued before the first conversion.
//
// FOR_ATTENTION: what a kernel reads that multiplies masked probabilities (zeros) with values.  A value of
// NaN would reach rows that do not see it; so a position whose key or value is NaN becomes a key of NaN
// with a value of zeros: its score is NaN for those who see it, and masked for the others.
// ------------------------------------------------------------------------------------------
struct ReadQ8Args {
    const uint8_t* k_codes;
    const uint8_t* v_codes;
    const float* k_scales;
    const float* v_scales;
    const int* page_table;
    int table_stride, out_stride, ring, n_pages;
    const int* seq_end;
    void* k_out;
    void* v_out;
    int rows, n_kv, hd;
    int fill;                      // 1: pages that hold nothing of their row are written as zeros too
    unsigned* status;
};

template <typename T> __device__ __forceinline__ void store16(T* p, const float* v);
template <> __device__ __forceinline__ void store16<float>(float* p, const float* v) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
template <> __device__ __forceinline__ void store16<__nv_bfloat16>(__nv_bfloat16* p, const float* v) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(p + 8) = make_uint4(w[4], w[5], w[6], w[7]);
}

#define RD_THREADS 256
template <typename T, int FMT, bool FOR_ATTENTION>
__global__ void __launch_bounds__(RD_THREADS) read_pages_q8_kernel(ReadQ8Args a) {
    pdl_launch_dependents();
    const int hk = blockIdx.y;
    const bool is_v = blockIdx.z != 0;
    const int row = blockIdx.x / a.out_stride, index = blockIdx.x - row * a.out_stride;
    const int end = a.seq_end[row];
    const int page = index < a.table_stride ? a.page_table[(long long)row * a.table_stride + index] : -1;
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
    const int upr = a.hd >> 4;                        // units a vector
    const int units = MF_PAGE * upr;
    const long long from = there ? ((long long)page * a.n_kv + hk) * MF_PAGE : 0;
    const uint8_t* codes = (is_v ? a.v_codes : a.k_codes) + from * a.hd;
    const float* scales = (is_v ? a.v_scales : a.k_scales) + from;
    const float* other = (is_v ? a.k_scales : a.v_scales) + from;
    T* out = (T*)(is_v ? a.v_out : a.k_out) + ((long long)blockIdx.x * a.n_kv + hk) * MF_PAGE * a.hd;
    for (int u0 = threadIdx.x; u0 < units; u0 += 2 * RD_THREADS) {
        uint4 w[2];
        float s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = u0 + i * RD_THREADS, place = u / upr;
            w[i] = make_uint4(0, 0, 0, 0);
            s[i] = 0.0f;
            if (u < units && place < n) {
                w[i] = *reinterpret_cast<const uint4*>(codes + (long long)u * 16);
                s[i] = scales[place];
                if (FOR_ATTENTION) {
                    const float so = other[place];
                    if (is_v && s[i] != s[i]) s[i] = 0.0f;
                    else if (!is_v && so != so) s[i] = so;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int u = u0 + i * RD_THREADS;
            if (u >= units) continue;
            const uint32_t words[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
            float v[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) q8_floats<FMT>(words[j], v + 4 * j);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] *= s[i];
            store16<T>(out + (long long)u * 16, v);
        }
    }
}

template <typename T, int FMT> static int read_launch(const ReadQ8Args& a, bool for_attention, cudaStream_t stream) {
    const dim3 grid((unsigned)(a.rows * a.out_stride), a.n_kv, 2);
    if (for_attention) mf_launch(read_pages_q8_kernel<T, FMT, true>, grid, dim3(RD_THREADS), 0, stream, a);
    else mf_launch(read_pages_q8_kernel<T, FMT, false>, grid, dim3(RD_THREADS), 0, stream, a);
    return MF_LAUNCH_CHECK();
}

extern "C" int mf_read_pages_q8(const void* k_codes, const void* v_codes, const float* k_scales, const float* v_scales,
                                const int* page_table, int table_stride, int out_stride, int ring, int n_pages,
                                const int* seq_end, void* k_out, void* v_out, int rows, int n_kv, int hd, int dtype,
                                int fmt, int fill, int for_attention, unsigned* status, cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (hd % 16 != 0 || hd < 16 || hd > 256 || n_kv <= 0 || n_kv > 65535) return MF_ERR_UNSUPPORTED;
    if (ring < 0 || ring % MF_PAGE != 0 || table_stride <= 0 || out_stride < table_stride || n_pages <= 0)
        return MF_ERR_ARGUMENT;
    if ((long long)rows * out_stride > 0x7fffffffLL || table_stride > 0x7fffffff / MF_PAGE) return MF_ERR_UNSUPPORTED;
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15) return MF_ERR_UNSUPPORTED;
    if ((dtype != MF_DTYPE_F32 && dtype != MF_DTYPE_BF16) || (fmt != MF_Q8_E4M3 && fmt != MF_Q8_INT8))
        return MF_ERR_UNSUPPORTED;
    ReadQ8Args a{};
    a.k_codes = (const uint8_t*)k_codes; a.v_codes = (const uint8_t*)v_codes; a.k_scales = k_scales;
    a.v_scales = v_scales; a.page_table = page_table; a.table_stride = table_stride; a.out_stride = out_stride;
    a.ring = ring; a.n_pages = n_pages; a.seq_end = seq_end; a.k_out = k_out; a.v_out = v_out; a.rows = rows;
    a.n_kv = n_kv; a.hd = hd; a.fill = fill; a.status = status;
    if (dtype == MF_DTYPE_F32)
        return fmt == MF_Q8_E4M3 ? read_launch<float, MF_Q8_E4M3>(a, for_attention != 0, stream)
                                 : read_launch<float, MF_Q8_INT8>(a, for_attention != 0, stream);
    return fmt == MF_Q8_E4M3 ? read_launch<__nv_bfloat16, MF_Q8_E4M3>(a, for_attention != 0, stream)
                             : read_launch<__nv_bfloat16, MF_Q8_INT8>(a, for_attention != 0, stream);
}
