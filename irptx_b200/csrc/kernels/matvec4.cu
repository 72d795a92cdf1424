// matvec4.cu -- y[m, n] = sum_k x[m, k] * s[n, k / group] * (q[n, k] - z[n, k / group]) with 4-bit
// weights q (two to a byte, the even k in the low half), group scales s and zero points z (8 when
// there are none), for a few tokens m.
//
// Bound: the packed weights are read once, half a byte each for 2 m operations, so HBM bounds it
// up to m of a few hundred; a call of a few megabytes is bound by latency.
//
// The products run on matrix instructions with the weights as the wide operand (16 rows of w) and
// the tokens as the narrow one (8). A weight becomes the exact bf16 number q - z: the
// four bits placed in the mantissa of 128 give 128 + q, from which 128 + z is subtracted. So no
// weight is rounded; a group's products are summed in f32 and the scale is applied to that sum.
// Which k an operand slot stands for does not matter as long as both operands agree, so each lane
// keeps the order in which its bytes come (k0 with k4, k1 with k5, ...), and the tokens are
// paired the same way with byte permutes.
#pragma once
#include "decode.cu"

#define MV4_WARPS 8

// 8 weights of one row: pairs (0, 4), (1, 5), (2, 6), (3, 7) minus the zero point pair.
__device__ __forceinline__ void mv4_unpack(uint32_t w, __nv_bfloat162 z, uint32_t (&r)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t u = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&u), z);
        r[i] = *reinterpret_cast<const uint32_t *>(&d);
    }
}

template <int B> struct mv4_vec;
template <> struct mv4_vec<16> { using T = uint4; };
template <> struct mv4_vec<8> { using T = uint2; };
template <> struct mv4_vec<4> { using T = unsigned; };

// GV: weights that share a scale, as far as the kernel is concerned (128, 64 or 32; group is a
// multiple of it). A warp's step is 128 weights of 16 RT rows: in each GV-wide piece the four lanes
// of a row take GV/4 weights each, so that one instruction never mixes two groups.
template <int GV, int RT>
struct Mv4Step {
    static constexpr int P = 128 / GV, WB = GV / 8;      // pieces; bytes of a lane's load
    typename mv4_vec<WB>::T w[RT][2][P];
    float s[RT][2];                                      // this lane's piece's scale (piece t * P / 4)
    unsigned z[RT][2];
};

template <int GV, int RT, bool Z>
__device__ __forceinline__ void mv4_load(const irx_kmv4_t &p, int64_t row0, int64_t kb, int g, int t, Mv4Step<GV, RT> &S)
{
    using St = Mv4Step<GV, RT>;
    using V = typename mv4_vec<St::WB>::T;
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int64_t row = row0 + rt * 16 + h * 8 + g;
            const bool in = row < p.n1;
            const uint8_t *w = p.w + row * p.w_stride;
#pragma unroll
            for (int i = 0; i < St::P; i++) {
                const int64_t k = kb * 128 + i * GV + t * (GV / 4);
                V v{};
                if (in && k < p.k) v = __ldcs(reinterpret_cast<const V *>(w + k / 2));
                S.w[rt][h][i] = v;
            }
            const int64_t ks = kb * 128 + (t * St::P / 4) * GV;
            float s = 0.0f;
            unsigned z = 8;
            if (in && ks < p.k) {
                const int64_t e = row * p.groups + (uint32_t)ks / (uint32_t)p.group;
                s = irx_ld1(p.s, p.sdt, e);
                if (Z) z = p.z[e];
            }
            S.s[rt][h] = s;
            S.z[rt][h] = z;
        }
}

template <int GV, int NT, int RT, bool Z>
__device__ __forceinline__ void mv4_step(const irx_kmv4_t &p, int64_t m0, int64_t kb, int g, int t,
                                         const Mv4Step<GV, RT> &S, float (&acc)[RT][NT][4])
{
    using St = Mv4Step<GV, RT>;
    constexpr int W = St::WB / 4;                        // words of a lane's load
    const int lane = g * 4 + t;
#pragma unroll
    for (int i = 0; i < St::P; i++) {
        float part[RT][NT][4];
        __nv_bfloat162 z[RT][2];
        float s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                unsigned zz = 8;
                if (St::P > 1) {
                    const int from = (lane & ~3) + i * 4 / St::P;
                    s[rt][h] = __shfl_sync(0xffffffffu, S.s[rt][h], from);
                    if (Z) zz = __shfl_sync(0xffffffffu, S.z[rt][h], from);
                } else {
                    s[rt][h] = S.s[rt][h];
                    if (Z) zz = S.z[rt][h];
                }
                const uint32_t zb = 0x43004300u | ((zz & 15u) * 0x00010001u);
                z[rt][h] = *reinterpret_cast<const __nv_bfloat162 *>(&zb);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) part[rt][nt][2 * h] = part[rt][nt][2 * h + 1] = 0.0f;
            }
#pragma unroll
        for (int w = 0; w < W; w++) {
            const int64_t k = kb * 128 + i * GV + t * (GV / 4) + w * 8;
            uint32_t b[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int64_t m = m0 + nt * 8 + g;
                uint4 x = make_uint4(0, 0, 0, 0);
                if (m < p.m && k < p.k)
                    x = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<const __nv_bfloat16 *>(p.x) + m * p.x_stride + k));
                b[nt][0] = __byte_perm(x.x, x.z, 0x5410);
                b[nt][1] = __byte_perm(x.x, x.z, 0x7632);
                b[nt][2] = __byte_perm(x.y, x.w, 0x5410);
                b[nt][3] = __byte_perm(x.y, x.w, 0x7632);
            }
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                uint32_t lo[4], hi[4];
                mv4_unpack(reinterpret_cast<const uint32_t *>(&S.w[rt][0][i])[w], z[rt][0], lo);
                mv4_unpack(reinterpret_cast<const uint32_t *>(&S.w[rt][1][i])[w], z[rt][1], hi);
                const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    mma_16816(part[rt][nt], a0, b[nt][0], b[nt][1]);
                    mma_16816(part[rt][nt], a1, b[nt][2], b[nt][3]);
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; rt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[rt][nt][j] = fmaf(s[rt][j >> 1], part[rt][nt][j], acc[rt][nt][j]);
    }
}

template <int GV, int NT, int RT, bool Z>
__device__ __forceinline__ void mv4_body(const irx_kmv4_t &p)
{
    __shared__ float red[MV4_WARPS][RT * 16][NT * 8 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int64_t nb = (p.n1 - p.n0 + RT * 16 - 1) / (RT * 16);
    const int64_t row0 = p.n0 + (blockIdx.x % nb) * (RT * 16), m0 = (blockIdx.x / nb) * (NT * 8);
    const int64_t steps = (p.k + 127) / 128;
    float acc[RT][NT][4];
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[rt][nt][j] = 0.0f;
    irx_pdl_enter();
    // the warps take the row's steps in turn, so neighbours read neighbouring bytes; a step's bytes are
    // loaded two steps ahead of their use
    Mv4Step<GV, RT> S[2];
    int64_t kb = warp;
    mv4_load<GV, RT, Z>(p, row0, kb, g, t, S[0]);
    mv4_load<GV, RT, Z>(p, row0, kb + MV4_WARPS, g, t, S[1]);
    for (; kb < steps; kb += 2 * MV4_WARPS) {
        mv4_step<GV, NT, RT, Z>(p, m0, kb, g, t, S[0], acc);
        mv4_load<GV, RT, Z>(p, row0, kb + 2 * MV4_WARPS, g, t, S[0]);
        if (kb + MV4_WARPS >= steps) break;
        mv4_step<GV, NT, RT, Z>(p, m0, kb + MV4_WARPS, g, t, S[1], acc);
        mv4_load<GV, RT, Z>(p, row0, kb + 3 * MV4_WARPS, g, t, S[1]);
    }
#pragma unroll
    for (int rt = 0; rt < RT; rt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) red[warp][rt * 16 + g + (j >> 1) * 8][nt * 8 + 2 * t + (j & 1)] = acc[rt][nt][j];
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 16 * NT * 8; i += MV4_WARPS * 32) {
        const int r = i % (RT * 16), c = i / (RT * 16);
        if (row0 + r >= p.n1 || m0 + c >= p.m) continue;
        float v = red[0][r][c];
#pragma unroll
        for (int w = 1; w < MV4_WARPS; w++) v += red[w][r][c];
        irx_st1(p.y, p.dt, (m0 + c) * p.n + row0 + r, v);
    }
}

// Any sizes, strides and types: a warp per row of w and four tokens, two weights a lane and step.
__device__ __forceinline__ void mv4_any_body(const irx_kmv4_t &p)
{
    const int lane = threadIdx.x & 31;
    const int64_t nb = p.n1 - p.n0, mb = (p.m + 3) / 4;
    irx_pdl_enter();
    for (int64_t u = (int64_t)blockIdx.x * MV4_WARPS + (threadIdx.x >> 5); u < nb * mb; u += (int64_t)gridDim.x * MV4_WARPS) {
        const int64_t row = p.n0 + u % nb, m0 = (u / nb) * 4;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t k = 2 * lane; k < p.k; k += 64) {
            const unsigned byte = p.w[row * p.w_stride + k / 2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (k + h >= p.k) break;
                const int64_t e = row * p.groups + (k + h) / p.group;
                const int z = p.z ? (p.z[e] & 15) : 8;
                const float w = (float)((int)((byte >> (4 * h)) & 15u) - z) * irx_ld1(p.s, p.sdt, e);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (m0 + i < p.m) acc[i] = fmaf(w, irx_ld1(p.x, p.dt, (m0 + i) * p.x_stride + k + h), acc[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v = acc[i];
#pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
            if (lane == 0 && m0 + i < p.m) irx_st1(p.y, p.dt, (m0 + i) * p.n + row, v);
        }
    }
}

#define MV4_K(GV, NT, RT) \
    extern "C" __global__ void __launch_bounds__(MV4_WARPS * 32) irx_mv4_##GV##_##NT(const __grid_constant__ irx_kmv4_t p) \
    { mv4_body<GV, NT, RT, false>(p); } \
    extern "C" __global__ void __launch_bounds__(MV4_WARPS * 32) irx_mv4z_##GV##_##NT(const __grid_constant__ irx_kmv4_t p) \
    { mv4_body<GV, NT, RT, true>(p); }

MV4_K(32, 1, 1) MV4_K(32, 2, 2) MV4_K(64, 1, 1) MV4_K(64, 2, 2) MV4_K(128, 1, 1) MV4_K(128, 2, 2)
extern "C" __global__ void __launch_bounds__(MV4_WARPS * 32) irx_mv4_any(const __grid_constant__ irx_kmv4_t p) { mv4_any_body(p); }
