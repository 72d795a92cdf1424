// rope.cu -- rotary positions, alone and on the way into a paged cache.
//
// y = a R(pos f) x on the rotated part of each head, the rest copied: a pair (x1, x2) turns to
// (x1 cos - x2 sin, x1 sin + x2 cos). Pairs are (i, i + pairs) or, interleaved, (2 i, 2 i + 1).
// Angles: position times frequency in 64 bits, counted in turns, so that the whole turns drop out
// exactly and what is left, below half a turn, has an error under 2^-22 of a turn for 2^31 positions of
// a frequency of one radian. Sine and cosine are f32 of that remainder (its f32 rounding put back to
// first order), products f32, one rounding to the output's type.
//
// Bound by HBM for large calls (floor: every row read once and written once) and by its chain
// of dependent loads for small ones. A warp takes a part of a token: first its rows' loads are
// issued, then the token's angles go to shared memory, one pair a lane, and every row reads them
// from there; queries, keys and values of a cache append are one list of rows. When a row's items divide a warp
// (heads of 64, 128, 256) a lane keeps its item's angles in registers instead and needs no division: 16381 tokens of
// 40 heads of 128 (bf16) 66.5 -> 56.1 us, 5.98 TB/s.
#pragma once
#include "common.cuh"

#define ROPE_WARPS 4
#define ROPE_UNROLL 4

template <class T, int V> struct rope_vec;
template <> struct rope_vec<__nv_bfloat16, 8> {
    uint4 r;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { r = __ldcs(reinterpret_cast<const uint4 *>(p)); }
    __device__ __forceinline__ void store(__nv_bfloat16 *p) const { __stcs(reinterpret_cast<uint4 *>(p), r); }
    __device__ __forceinline__ void get(float (&o)[8]) const
    {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            o[2 * i] = __uint_as_float(w[i] << 16);
            o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&o)[8])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(o[2 * i], o[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
        r = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct rope_vec<float, 4> {
    float4 r;
    __device__ __forceinline__ void load(const float *p) { r = __ldcs(reinterpret_cast<const float4 *>(p)); }
    __device__ __forceinline__ void store(float *p) const { __stcs(reinterpret_cast<float4 *>(p), r); }
    __device__ __forceinline__ void get(float (&o)[4]) const { o[0] = r.x; o[1] = r.y; o[2] = r.z; o[3] = r.w; }
    __device__ __forceinline__ void set(const float (&o)[4]) { r = make_float4(o[0], o[1], o[2], o[3]); }
};
template <class T> struct rope_vec<T, 1> {
    T r;
    __device__ __forceinline__ void load(const T *p) { r = *p; }
    __device__ __forceinline__ void store(T *p) const { *p = r; }
    __device__ __forceinline__ void get(float (&o)[1]) const { o[0] = (float)r; }
    __device__ __forceinline__ void set(const float (&o)[1]) { r = (T)o[0]; }
};

// FIXED: a row's items divide 32, so that a lane has the same one of every row that it takes.
template <class T, int V, bool FIXED>
__device__ __forceinline__ void rope_body(const irx_krope_t &p)
{
    irx_pdl_enter();
    __shared__ float2 angles[ROPE_WARPS][128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t w = (int64_t)blockIdx.x * ROPE_WARPS + warp, t = p.t0 + w / p.parts;
    if (t >= p.t1) return;
    const int pos = p.pos[t];
    if (pos < 0) return;                                 // padding
    const int all = (p.heads + 2 * p.kv) * p.items, rotated = p.pairs / V;
    const int begin = (int)(w % p.parts) * p.chunk, end = min(all, begin + p.chunk);
    const T *q = reinterpret_cast<const T *>(p.q) + t * p.x_stride;
    const T *kn = reinterpret_cast<const T *>(p.kn) + t * p.kv_stride, *vn = reinterpret_cast<const T *>(p.vn) + t * p.kv_stride;
    T *qo = reinterpret_cast<T *>(p.qo) + t * p.y_stride;
    int64_t slot = -1;                                   // the token's first element in the pools, once known
    float2 *cs = angles[warp], own[V];
    const int per = FIXED ? 32 / p.items : 0, my_row = FIXED ? lane / p.items : 0, my_item = FIXED ? lane - my_row * p.items : 0;

    for (int i0 = begin; i0 < end; i0 += 32 * ROPE_UNROLL) {
        rope_vec<T, V> a[ROPE_UNROLL], b[ROPE_UNROLL];
        int row[ROPE_UNROLL], item[ROPE_UNROLL];
#pragma unroll
        for (int u = 0; u < ROPE_UNROLL; u++) {
            const int e = i0 + 32 * u + lane;
            row[u] = -1;
            if (e >= end) continue;
            const int r = FIXED ? ((i0 >> 5) + u) * per + my_row : e / p.items, j = FIXED ? my_item : e - r * p.items;
            row[u] = r;
            item[u] = j;
            const T *src = r < p.heads ? q + r * p.d : r < p.heads + p.kv ? kn + (r - p.heads) * p.d : vn + (r - p.heads - p.kv) * p.d;
            const int e0 = p.inter || j >= rotated ? 2 * j * V : j * V, e1 = p.inter || j >= rotated ? e0 + V : e0 + p.pairs;
            a[u].load(src + e0);
            if (e1 < p.d) b[u].load(src + e1);           // (a copied row's end may be half an item)
        }
        if (i0 == begin) {
            if (p.kv) {
                const int seq = p.seq[t], pi = pos / p.page_size;
                int64_t page = -1;
                if (seq >= 0 && seq < p.batch && pi < p.cols) page = p.table[(int64_t)seq * p.cols + pi];
                if (page >= 0 && page < p.pages) slot = page * p.page_stride + (int64_t)(pos - pi * p.page_size) * p.token_stride;
                else if (lane == 0) atomicOr(p.err, IRX_KERR_INDEX);
            }
            for (int f = lane; f < p.pairs; f += 32) {
                const double turns = (double)pos * p.freq[f], part = turns - rint(turns);
                const float hi = (float)part, lo = (float)(part - (double)hi) * 6.283185307f;
                float s, c;
                sincospif(2.0f * hi, &s, &c);
                cs[f] = make_float2((c - s * lo) * p.amp, (s + c * lo) * p.amp);
            }
            __syncwarp();
            if (FIXED && my_item < rotated)
#pragma unroll
                for (int i = 0; i < V; i++) own[i] = cs[my_item * V + i];
        }
#pragma unroll
        for (int u = 0; u < ROPE_UNROLL; u++) {
            if (row[u] < 0) continue;
            const int r = row[u], j = item[u];
            T *dst;
            if (r < p.heads) {
                dst = qo + r * p.d;
            } else {
                if (slot < 0) continue;                  // no such page: reported above
                dst = r < p.heads + p.kv ? reinterpret_cast<T *>(p.k) + slot + (int64_t)(r - p.heads) * p.head_stride
                                         : reinterpret_cast<T *>(p.v) + slot + (int64_t)(r - p.heads - p.kv) * p.head_stride;
            }
            if (r < p.heads + p.kv && j < rotated) {
                float x[V], y[V];
                a[u].get(x);
                b[u].get(y);
                if (V > 1 && p.inter) {
#pragma unroll
                    for (int i = 0; i < V / 2; i++) {
                        const float2 g = FIXED ? own[i] : cs[j * V + i], h = FIXED ? own[V / 2 + i] : cs[j * V + V / 2 + i];
                        const float x0 = x[2 * i], x1 = x[2 * i + 1], y0 = y[2 * i], y1 = y[2 * i + 1];
                        x[2 * i] = x0 * g.x - x1 * g.y;
                        x[2 * i + 1] = x0 * g.y + x1 * g.x;
                        y[2 * i] = y0 * h.x - y1 * h.y;
                        y[2 * i + 1] = y0 * h.y + y1 * h.x;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; i++) {
                        const float2 g = FIXED ? own[i] : cs[j * V + i];
                        const float x0 = x[i], x1 = y[i];
                        x[i] = x0 * g.x - x1 * g.y;
                        y[i] = x0 * g.y + x1 * g.x;
                    }
                }
                a[u].set(x);
                b[u].set(y);
            }
            const int e0 = p.inter || j >= rotated ? 2 * j * V : j * V, e1 = p.inter || j >= rotated ? e0 + V : e0 + p.pairs;
            a[u].store(dst + e0);
            if (e1 < p.d) b[u].store(dst + e1);
        }
    }
}

extern "C" __global__ void __launch_bounds__(128) irx_rope_bf16_lane(const __grid_constant__ irx_krope_t p) { rope_body<__nv_bfloat16, 8, true>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_rope_bf16_8(const __grid_constant__ irx_krope_t p) { rope_body<__nv_bfloat16, 8, false>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_rope_bf16_1(const __grid_constant__ irx_krope_t p) { rope_body<__nv_bfloat16, 1, false>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_rope_f32_lane(const __grid_constant__ irx_krope_t p) { rope_body<float, 4, true>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_rope_f32_4(const __grid_constant__ irx_krope_t p) { rope_body<float, 4, false>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_rope_f32_1(const __grid_constant__ irx_krope_t p) { rope_body<float, 1, false>(p); }
