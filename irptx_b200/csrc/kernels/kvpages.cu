// kvpages.cu -- the paged cache's data movement: new tokens into their pages, and page copies
// (forks that are written to, compaction).
//
// Both only move bytes, so they are bound by HBM for large calls (floor: the moved bytes read once
// and written once) and by the launch and the chain of dependent loads for small ones. They are
// written on vectors of 16, 4 or 2 bytes: the launcher takes the widest that every base and
// stride allows. Measured: 16,376 tokens of 8 heads of 128 (bf16, 125 MB moved) appended in 21.4 us,
// 5.8 TB/s; 1023 pages of 32 KB in 4 layers and 2 pools (536 MB moved) copied in 86 us, 6.2 TB/s;
// the smallest calls 2.0 and 2.4 us, about an empty launch.
#pragma once
#include "common.cuh"

__device__ __forceinline__ void irx_flag(unsigned *err, unsigned bit)
{
    atomicOr(err, bit);
}

// ---- append ----
// One warp moves up to APP_VEC x 32 vectors of a token's keys and as many of its values. The data loads
// are issued before the token's slot is known (sequence and position, then the page table): only
// the stores wait for that chain. Two vectors of each a lane: one token of 8 heads of 128 is then two
// warps (0.2 us less for 32 tokens than four vectors, one warp; long calls do not change).
#define APP_VEC IRX_APPEND_VEC

template <class V>
__device__ __forceinline__ void append_body(const irx_kapp_t &p)
{
    irx_pdl_enter();
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    const int64_t t = p.t0 + w / p.parts;
    if (t >= p.t1) return;
    const int part = (int)(w % p.parts), row = p.heads * p.dv;
    const int e0 = part * (32 * APP_VEC) + lane;
    const int pos = p.pos[t], seq = p.seq[t];
    if (pos < 0) return;                                 // padding
    const V *kn = reinterpret_cast<const V *>(p.kn) + t * p.stride, *vn = reinterpret_cast<const V *>(p.vn) + t * p.stride;
    V a[APP_VEC], b[APP_VEC];
#pragma unroll
    for (int i = 0; i < APP_VEC; i++) {
        const int e = e0 + 32 * i;
        if (e < row) {
            a[i] = __ldcs(kn + e);
            b[i] = __ldcs(vn + e);
        }
    }
    const int pi = pos / p.page_size, slot = pos - pi * p.page_size;
    int64_t page = -1;
    if (seq >= 0 && seq < p.batch && pi < p.cols) page = p.table[(int64_t)seq * p.cols + pi];
    if (page < 0 || page >= p.pages) {
        if (lane == 0) irx_flag(p.err, IRX_KERR_INDEX);
        return;
    }
    const int64_t base = page * p.page_stride + (int64_t)slot * p.token_stride;
    V *k = reinterpret_cast<V *>(p.k) + base, *v = reinterpret_cast<V *>(p.v) + base;
#pragma unroll
    for (int i = 0; i < APP_VEC; i++) {
        const int e = e0 + 32 * i;
        if (e < row) {
            const int h = e / p.dv;
            const int64_t o = (int64_t)h * p.head_stride + (e - h * p.dv);
            __stcs(k + o, a[i]);
            __stcs(v + o, b[i]);
        }
    }
}

extern "C" __global__ void __launch_bounds__(128) irx_kv_append_16(const __grid_constant__ irx_kapp_t p) { append_body<uint4>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_kv_append_4(const __grid_constant__ irx_kapp_t p) { append_body<unsigned>(p); }
extern "C" __global__ void __launch_bounds__(128) irx_kv_append_2(const __grid_constant__ irx_kapp_t p) { append_body<unsigned short>(p); }

// ---- page copy ----
// A block copies one tile, 256 threads x CPY_VEC vectors, of one page of one layer of one pool; all of
// a thread's loads are in flight before its first store. Two vectors a thread: 86 us for the 536 MB above;
// with four 92, with one 104.
#define CPY_THREADS 256
#define CPY_VEC (IRX_COPY_TILE / CPY_THREADS)

template <class V>
__device__ __forceinline__ void copy_body(const irx_kcpy_t &p)
{
    irx_pdl_enter();
    const int64_t per_pair = p.tiles * p.layers * 2, all = (p.p1 - p.p0) * per_pair;
    const int64_t page = p.run * p.n1 * p.n2;
    for (int64_t u = blockIdx.x; u < all; u += gridDim.x) {
        const int64_t pair = p.p0 + u / per_pair;
        int64_t r = u % per_pair;
        const int64_t tile = r % p.tiles;
        r /= p.tiles;
        const int layer = (int)(r >> 1);
        V *pool = reinterpret_cast<V *>(r & 1 ? p.v : p.k) + (int64_t)layer * p.layer_stride;
        const int64_t src = p.pairs[2 * pair], dst = p.pairs[2 * pair + 1];
        if (src < 0 && src == dst) continue;             // padding (-1, -1)
        if (src < 0 || dst < 0 || src >= p.pages || dst >= p.pages) {
            if (threadIdx.x == 0) irx_flag(p.err, IRX_KERR_INDEX);
            continue;
        }
        const V *s = pool + src * p.page_stride;
        V *d = pool + dst * p.page_stride;
        V a[CPY_VEC];
        int64_t o[CPY_VEC];
#pragma unroll
        for (int i = 0; i < CPY_VEC; i++) {
            const int64_t e = tile * (CPY_THREADS * CPY_VEC) + i * CPY_THREADS + threadIdx.x;
            o[i] = -1;
            if (e < page) {
                if (p.n1 == 1 && p.n2 == 1) o[i] = e;
                else {
                    const int64_t q = e / p.run, i2 = q / p.n1;
                    o[i] = (e - q * p.run) + (q - i2 * p.n1) * p.s1 + i2 * p.s2;
                }
                a[i] = __ldcs(s + o[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < CPY_VEC; i++)
            if (o[i] >= 0) __stcs(d + o[i], a[i]);
    }
}

extern "C" __global__ void __launch_bounds__(CPY_THREADS) irx_kv_copy_16(const __grid_constant__ irx_kcpy_t p) { copy_body<uint4>(p); }
extern "C" __global__ void __launch_bounds__(CPY_THREADS) irx_kv_copy_4(const __grid_constant__ irx_kcpy_t p) { copy_body<unsigned>(p); }
extern "C" __global__ void __launch_bounds__(CPY_THREADS) irx_kv_copy_2(const __grid_constant__ irx_kcpy_t p) { copy_body<unsigned short>(p); }
