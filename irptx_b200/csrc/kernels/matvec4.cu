// matvec4.cu -- y[m, n] = sum_k x[m, k] * s[n, k / group] * (q[n, k] - z[n, k / group]) with 4-bit
// weights q (two to a byte, the even k in the low half), group scales s and zero points z (8 when
// there are none), for a few tokens m.
//
// Bound: the packed weights are read, half a byte each for 2 m operations, so HBM sets the floor up to m of
// a few hundred. The kernel stays at a third of it, and no single part is why: of 27.8 us in an earlier
// build of the largest call below, 23.7 were left without the unpacking (4 logic operations, 3 shifts and
// 4 subtractions for 8 weights, whatever m is), 17.8 without the products, 13.7 with the weights'
// stream alone. A warp goes through a chain, unpack, then up to 8 products into one accumulator, and 16
// warps an SM are too few to cover it (0.46 instructions issue a cycle and scheduler, the matrix pipe is
// 24 % busy); equal slices also leave places empty (226 or 256 blocks where 296 fit). A call of a few
// megabytes is bound by latency. Measured, bf16: [13 x 14336] x [8192 x 14336] (61 MB) 24.2 us, 2.5 TB/s;
// [4 x 4096] x [14337 x 4096] with zero points 14.6 us; one token, 4096 x 4096, 6.0 us.
// More than 16 tokens (5 in f32) go over the weights again for each 16 (5): 17 tokens of the largest
// call take 42.2 us, 64 77.8, and 13 in f32 87 where 5 take 27.6.
//
// The products run on matrix instructions with the weights as the wide operand (16 rows of w) and
// the tokens as the narrow one (8). A weight becomes the exact bf16 number q - z (over 2^11): the
// four bits placed in the mantissa of 128 give 128 + q, from which 128 + z is subtracted. So no
// weight is rounded; a group's products are summed in f32 and the scale is applied to that sum.
// Which k an operand slot stands for does not matter as long as both operands agree, so each lane
// keeps the order in which its bytes come (k0 with k4, k1 with k5, ...), and the tokens are
// paired the same way with byte permutes. (tcgen05 with the unpacked weights in tensor memory as its
// A operand measured no better, 28 us against 26 at the first size and 8.9 against 5.8 at the last: the
// unpacking is the same work, and each chunk's hand-over to the one thread that issues products
// adds latency.)
#pragma once
#include <type_traits>
#include "decode.cu"

#define MV4_WARPS 8
// Two bf16 numbers of 128 / 2^11, whose last mantissa place is 1 / 2^11: the weights enter the products as
// (q - z) / 2^11, so that a group's sum, up to 15 * 128 tokens before its scale, stays in range for
// every finite token; 2^11 is given back with the last sum.
#define MV4_ONE 0x3d803d80u
#define MV4_BACK 2048.0f

// 8 weights of one row: pairs (0, 4), (1, 5), (2, 6), (3, 7) minus the zero point pair.
__device__ __forceinline__ void mv4_unpack(uint32_t w, __nv_bfloat162 z, uint32_t (&r)[4])
{
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t u;
        asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(u) : "r"(w), "r"(0x000f000fu), "r"(MV4_ONE));   // (w & m) | c
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&u), z);
        r[i] = *reinterpret_cast<const uint32_t *>(&d);
        w >>= 4;
    }
}

// The tiling. A block takes 128 rows of w and a slice of k, in stages of 256 k: 128 bytes of every
// row, with the tokens' values of those k, through a ring of asynchronous copies, so that bytes
// are in flight whatever the warps do. Its 8 warps are 4 groups of 32 rows times 2 halves of a
// stage. The weights of a stage come by one TMA copy, which also fills zeros past the ends and
// swizzles the 16-byte pieces for ldmatrix. The slices of k of the same rows are a cluster's blocks,
// which add up through distributed shared memory in a fixed order: that is how a matrix of few
// rows still fills the GPU, with no workspace and the same bits every time.
//
// A stage's 16 bytes of a row are 32 weights; ldmatrix hands lane (g, t) the 8 weights t of row g, so
// an instruction's four lanes always lie in one group of 32, whatever the group size is (GV: 128,
// 64 or 32, the widest that divides it).
//
// f32 tokens are carried as three bf16 columns each, high, middle and low part, whose sum is the
// f32 value to its last bit (unless that is below bf16's range): the same products, exact, and
// the three columns' sums are added at the end.
template <int NT>
struct Mv4Smem {
    // zero points: as the pairs that are subtracted where there is room, bytes with 16 columns
    using Zero = typename std::conditional<NT == 1, uint32_t, unsigned char>::type;
    static constexpr int ZB = (int)sizeof(Zero), ZS = NT == 1 ? 9 : 8;
    static constexpr int XS = 512 + 64;                  // bytes of a column's stage: 64 off the banks' period
    static constexpr int W = 128 * 128, X = NT * 8 * XS, RING = W * IRX_MV4_STAGES, SCALES = RING + X * IRX_MV4_STAGES;
    static constexpr int ZEROS = SCALES + 2 * 128 * 9 * 4, BARS = ZEROS + 2 * 128 * ZS * ZB;
    static_assert(BARS + 1024 + 64 == IRX_MV4_SMEM(NT), "the launcher's shared memory size");
    static constexpr int RS = NT * 8 + 4;                // floats of a row of the sums
    static_assert(2 * 128 * RS * 4 <= SCALES, "the sums fit the ring");
};

// The first product of a sum: the accumulators start at zero.
__device__ __forceinline__ void mma_16816_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

template <int GV, int NT>
__device__ __forceinline__ void mv4_stage(uint32_t ws, const unsigned char *xs, const float *sc, const typename Mv4Smem<NT>::Zero *zp, int wr, int wk, int lane,
                                          float (&acc)[2][NT][4])
{
    using M = Mv4Smem<NT>;
    constexpr int P = 128 / GV;                          // pieces of a warp's 128 k
    const int g = lane >> 2, t = lane & 3;
    uint32_t w[2][4];                                    // of two steps, both row tiles
#pragma unroll
    for (int i = 0; i < P; i++) {
        float part[2][NT][4];
        __nv_bfloat162 z[2][2];
        float s[2][2];
#pragma unroll
        for (int rt = 0; rt < 2; rt++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = wr * 32 + rt * 16 + h * 8 + g;
                uint32_t zb = MV4_ONE + 0x00080008u;     // a zero point of 8
                if (zp) {
                    zb = zp[row * M::ZS + i];
                    if (NT > 1) zb = MV4_ONE | ((zb & 15u) * 0x00010001u);
                }
                s[rt][h] = sc[row * 9 + i];
                z[rt][h] = *reinterpret_cast<const __nv_bfloat162 *>(&zb);
            }
#pragma unroll
        for (int q = 0; q < 4 / P; q++) {
            const int step = i * (4 / P) + q;
            if ((step & 1) == 0) {
#pragma unroll
                for (int rt = 0; rt < 2; rt++) {
                    const int row = wr * 32 + rt * 16 + (lane & 15), ch = wk * 4 + step + (lane >> 4);
                    ldsm4(w[rt], ws + row * 128 + ((ch ^ (row & 7)) << 4));
                }
            }
            uint32_t b[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint4 x = *reinterpret_cast<const uint4 *>(xs + (nt * 8 + g) * M::XS + (wk * 128 + step * 32 + t * 8) * 2);
                b[nt][0] = x.x;
                b[nt][1] = x.y;
                b[nt][2] = x.z;
                b[nt][3] = x.w;
            }
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                uint32_t lo[4], hi[4];
                mv4_unpack(w[rt][(step & 1) * 2], z[rt][0], lo);
                mv4_unpack(w[rt][(step & 1) * 2 + 1], z[rt][1], hi);
                const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if (q == 0) mma_16816_first(part[rt][nt], a0, b[nt][0], b[nt][1]);
                    else mma_16816(part[rt][nt], a0, b[nt][0], b[nt][1]);
                    mma_16816(part[rt][nt], a1, b[nt][2], b[nt][3]);
                }
            }
        }
#pragma unroll
        for (int rt = 0; rt < 2; rt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[rt][nt][j] = fmaf(s[rt][j >> 1], part[rt][nt][j], acc[rt][nt][j]);
    }
}

// Four floats of any block of the cluster; not volatile, so that several can be on their way at once (the
// cluster barriers on both sides are).
__device__ __forceinline__ float4 ld_cluster4(uint32_t a)
{
    float4 x;
    asm("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(a));
    return x;
}

template <int GV, int NT, bool F32>
__device__ __forceinline__ void mv4_body(const irx_kmv4_t &p)
{
    using M = Mv4Smem<NT>;
    extern __shared__ unsigned char sm_raw[];
    unsigned char *sm = sm_raw + ((1024u - (irx_smem_u32(sm_raw) & 1023u)) & 1023u);   // the swizzle's period
    constexpr int ST = IRX_MV4_STAGES, COLS = NT * 8, TOK = F32 ? COLS / 3 : COLS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wr = warp & 3, wk = warp >> 2, g = lane >> 2, t = lane & 3;
    const int ck = p.ck, rank = (int)(blockIdx.x % (unsigned)ck);
    const unsigned tile = blockIdx.x / (unsigned)ck, nb = (unsigned)((p.n1 - p.n0 + 127) >> 7), mt = nb == 1 ? tile : tile / nb;
    const int row0 = (int)p.n0 + (int)(tile - mt * nb) * 128, n1 = (int)p.n1, m0 = (int)mt * TOK, m_all = (int)p.m;
    // this block's stages: rank, rank + ck, ..., so that the cluster reads neighbouring bytes of a row at a time
    const int k_all = (int)p.k, steps = (k_all + 255) >> 8, n_st = (steps - rank + ck - 1) / ck;
    float acc[2][NT][4];
#pragma unroll
    for (int rt = 0; rt < 2; rt++)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[rt][nt][j] = 0.0f;
    uint64_t *full = reinterpret_cast<uint64_t *>(sm + M::BARS);
    if (tid == 0) {
        for (int i = 0; i < ST; i++) irx_mbar_init(full + i, 1);
        irx_fence_mbar_init();
        tma_prefetch_desc(&p.tma_w);
    }
    irx_pdl_enter();
    __syncthreads();

    auto fetch = [&](int s, int slot) {                  // stage s into its slot, by one thread
        if (tid == 0 && s < n_st) {
            irx_mbar_expect_tx(full + slot, M::W);
            tma_load_2d(sm + slot * M::W, &p.tma_w, (s * ck + rank) * 128, row0, full + slot);
        }
    };
    // The tokens' part, a stage ahead in registers, stored in the order in which the weights unpack: bf16 8
    // k of columns tid / 32 + 8 i at a time, f32 the stage's k = tid of every token, in three parts
    // (truncations, so that the parts of an infinity or a NaN stay what they should).
    uint4 xb[F32 ? 1 : NT];
    float xr[F32 ? TOK : 1];
    const char *xsrc = reinterpret_cast<const char *>(p.x) +
        (F32 ? ((int64_t)m0 * p.x_stride + tid + rank * 256) * 4 : ((int64_t)(m0 + (tid >> 5)) * p.x_stride + (tid & 31) * 8 + rank * 256) * 2);
    const int64_t xrow = p.x_stride * (F32 ? 4 : 16), xadv = (int64_t)ck * 256 * (F32 ? 4 : 2);
    int xk = rank * 256 + (F32 ? tid : (tid & 31) * 8);   // the k that the next load starts at
    const int xleft = m_all - m0 - (F32 ? 0 : tid >> 5);
    auto xload = [&]() {
        const bool kin = xk < k_all;
        if (F32) {
#pragma unroll
            for (int m = 0; m < TOK; m++) {
                xr[m] = 0.0f;
                if (kin && m < xleft) xr[m] = __ldg(reinterpret_cast<const float *>(xsrc + m * xrow));
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; i++) {
                xb[i] = make_uint4(0, 0, 0, 0);
                if (kin && 8 * i < xleft) xb[i] = __ldg(reinterpret_cast<const uint4 *>(xsrc + i * xrow));
            }
        }
        xk += ck * 256;
        xsrc += xadv;
    };
    auto xstore = [&](int slot) {
        unsigned char *st = sm + M::RING + slot * M::X;
        if (F32) {
            const int k8 = tid & 7;
            st += ((tid & ~7) + (k8 < 4 ? 2 * k8 : 2 * k8 - 7)) * 2;
#pragma unroll
            for (int m = 0; m < TOK; m++) {
                const __nv_bfloat16 hi = __float2bfloat16_rz(xr[m]);
                const float r1 = isinf(xr[m]) ? 0.0f : xr[m] - __bfloat162float(hi);
                const __nv_bfloat16 mid = __float2bfloat16_rz(r1);
                const __nv_bfloat16 lo = __float2bfloat16_rz(r1 - __bfloat162float(mid));
                *reinterpret_cast<__nv_bfloat16 *>(st + (3 * m) * M::XS) = hi;
                *reinterpret_cast<__nv_bfloat16 *>(st + (3 * m + 1) * M::XS) = mid;
                *reinterpret_cast<__nv_bfloat16 *>(st + (3 * m + 2) * M::XS) = lo;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NT; i++)
                *reinterpret_cast<uint4 *>(st + ((tid >> 5) + 8 * i) * M::XS + (tid & 31) * 16) =
                    make_uint4(__byte_perm(xb[i].x, xb[i].z, 0x5410), __byte_perm(xb[i].x, xb[i].z, 0x7632),
                               __byte_perm(xb[i].y, xb[i].w, 0x5410), __byte_perm(xb[i].y, xb[i].w, 0x7632));
        }
    };
    // Scales and zero points: 8 pieces of GV k a row serve a run of 4, 2 or 1 stages. A thread loads four
    // pieces, eight neighbouring threads a row's, a run ahead in registers (as they lie in memory), and
    // stores them as numbers when the run before them is done with: every lane loading its own rows'
    // each stage took as long as half the products.
    constexpr int P = 128 / GV, RUN = 4 / P;
    float *scales = reinterpret_cast<float *>(sm + M::SCALES);
    typename M::Zero *zeros = reinterpret_cast<typename M::Zero *>(sm + M::ZEROS);
    uint32_t sr[4], zr[4];
    uint32_t at[4];                                      // rows past the end read the last row's: their sums go nowhere
#pragma unroll
    for (int i = 0; i < 4; i++) at[i] = (uint32_t)min(row0 + (tid >> 3) + 32 * i, n1 - 1) * (uint32_t)p.groups;
    auto sload = [&](int r) {                            // run r; k / 32 / (group / 32) is a multiplication, exact below 2^26
        const int pc = tid & 7;
        const uint32_t k = min((uint32_t)(((r * RUN + pc / (2 * P)) * ck + rank) * 256 + (pc % (2 * P)) * GV), (uint32_t)k_all - 1);
        const uint32_t grp = (uint32_t)(((uint64_t)(k >> 5) * p.gmul) >> p.gshift);
        if (p.sdt == DT_BF16) {
#pragma unroll
            for (int i = 0; i < 4; i++) sr[i] = __ldg(reinterpret_cast<const unsigned short *>(p.s) + (at[i] + grp));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) sr[i] = __ldg(reinterpret_cast<const uint32_t *>(p.s) + (at[i] + grp));
        }
        if (p.z) {
#pragma unroll
            for (int i = 0; i < 4; i++) zr[i] = __ldg(p.z + (at[i] + grp));
        }
    };
    auto sstore = [&](int r) {
        const int shift = p.sdt == DT_BF16 ? 16 : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int row = (r & 1) * 128 + (tid >> 3) + 32 * i;
            scales[row * 9 + (tid & 7)] = __uint_as_float(sr[i] << shift);
            if (p.z) zeros[row * M::ZS + (tid & 7)] = (typename M::Zero)(NT == 1 ? MV4_ONE | ((zr[i] & 15u) * 0x00010001u) : zr[i]);
        }
    };
    if (F32) {                                           // columns that no token has stay zero
        for (int i = tid; i < ST * M::X / 16; i += MV4_WARPS * 32) *reinterpret_cast<uint4 *>(sm + M::RING + i * 16) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < ST - 1; i++) fetch(i, i);
    sload(0);
    xload();
    sstore(0);
    sload(1);
    xstore(0);
    xload();
    int ok = 1;
    int slot = 0;
    unsigned phase = 0;
    for (int c = 0; c < n_st; c++) {
        const int run = c / RUN, sub = c % RUN, next = slot + 1 == ST ? 0 : slot + 1;
        ok = ok && irx_mbar_wait(full + slot, phase);
        __syncthreads();                                 // tokens and scales are there too; the stage before is free
        fetch(c + ST - 1, slot ? slot - 1 : ST - 1);
        mv4_stage<GV, NT>(irx_smem_u32(sm) + slot * M::W, sm + M::RING + slot * M::X,
                          scales + (run & 1) * (128 * 9) + sub * (2 * P) + wk * P,
                          p.z ? zeros + (run & 1) * (128 * M::ZS) + sub * (2 * P) + wk * P : nullptr, wr, wk, lane, acc);
        if (c + 1 < n_st) {
            if (sub == RUN - 1) {
                sstore(run + 1);
                sload(run + 2);
            }
            xstore(next);
            xload();
        }
        slot = next;
        phase ^= next == 0;
    }
    if (!ok) {                                           // a wait ran out: report it, and let copies in flight land
        irx_flag(p.err, IRX_KERR_TIMEOUT);
        for (int s = max(0, n_st - ST); s < n_st; s++) irx_mbar_wait(full + s % ST, (s / ST) & 1);
    }
    __syncthreads();
    // the second half's sums go through shared memory to the first half's warps, which leave the block's
    // 128 x COLS sums there; then every block of the cluster adds up its share of the rows
    float *red = reinterpret_cast<float *>(sm);
#pragma unroll
    for (int half = 1; half >= 0; half--) {
        if (wk == half) {
#pragma unroll
            for (int rt = 0; rt < 2; rt++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float *a = red + (wr * 32 + rt * 16 + g + (j >> 1) * 8) * M::RS + nt * 8 + 2 * t + (j & 1);
                        *a = half ? acc[rt][nt][j] : acc[rt][nt][j] + *a;
                    }
        }
        if (half) __syncthreads();
    }
    if (ck > 1) cluster_sync(); else __syncthreads();
    const int r0 = rank * ((127 + ck) / ck), rows = min((127 + ck) / ck, 128 - r0);   // (not below 0: ck is 8 at most)
    const float *fin = red + r0 * M::RS;
    if (ck > 1) {
        float *sum = red + 128 * M::RS;
        for (int i = tid; i < rows * (COLS / 4); i += MV4_WARPS * 32) {
            const int r = i / (COLS / 4), c = (i % (COLS / 4)) * 4;
            const float *a = red + (r0 + r) * M::RS + c;
            float4 v = ld_cluster4(cluster_addr(a, 0));
            for (int q = 1; q < ck; q++) {
                const float4 x = ld_cluster4(cluster_addr(a, q));
                v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            }
            *reinterpret_cast<float4 *>(sum + r * M::RS + c) = v;
        }
        __syncthreads();
        fin = sum;
    }
    for (int i = tid; i < rows * TOK; i += MV4_WARPS * 32) {
        const int m = i / rows, r = i - m * rows;
        const float *a = fin + r * M::RS + (F32 ? 3 * m : m);
        const float v = F32 ? a[0] + (a[1] + a[2]) : a[0];
        if (row0 + r0 + r < n1 && m0 + m < m_all) irx_st1(p.y, p.dt, (int64_t)(m0 + m) * p.n + row0 + r0 + r, v * MV4_BACK);
    }
    if (ck > 1) cluster_sync();                        // no block leaves while its sums are still read
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

#define MV4_K(GV, NT) \
    extern "C" __global__ void __launch_bounds__(MV4_WARPS * 32, 2) irx_mv4_bf16_##GV##_##NT(const __grid_constant__ irx_kmv4_t p) \
    { mv4_body<GV, NT, false>(p); } \
    extern "C" __global__ void __launch_bounds__(MV4_WARPS * 32, 2) irx_mv4_f32_##GV##_##NT(const __grid_constant__ irx_kmv4_t p) \
    { mv4_body<GV, NT, true>(p); }

MV4_K(32, 1) MV4_K(32, 2) MV4_K(64, 1) MV4_K(64, 2) MV4_K(128, 1) MV4_K(128, 2)
extern "C" __global__ void __launch_bounds__(MV4_WARPS * 32) irx_mv4_any(const __grid_constant__ irx_kmv4_t p) { mv4_any_body(p); }
