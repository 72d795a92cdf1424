// prompt_tc.cu -- attention over packed prompts on the 5th-generation tensor cores: bf16, head sizes up to 128
// in multiples of 8, up to 128 query heads a key-value head.
//
// A unit is two 128-row tiles of one (sequence, key-value head): tp = 128 / group tokens each with all
// their heads, loaded as one box of the queries (64 columns, group, 1, tp). Keys and values come in tiles of
// 128 tokens, boxes that begin at any row; columns past the head size are filled with zeros by the
// copy. The pipeline is irx_attn_bf16's (attn.cu): scores S_t = Q_t K^T into TMEM, one thread a row for the softmax,
// P over the scores' columns, O_t += P_t V, each tile's softmax under the other tile's products. What differs:
//   * warp 8 finds the block's units from `starts` (prompt.cu) and hands them out with the loads;
//   * key tiles may begin anywhere and are masked by token: a window's edge and the sinks' tiles too. With heads above 64
//     the sinks' tile and a unit's last one are 64 keys wide when that holds all that is seen of them;
//   * warps 10 and 11 look through the values of the tiles that a mask cuts. Rows that no query of the unit
//     sees become zeros, for another sequence's numbers or uninitialised ones may lie there and 0 * NaN is NaN.
//     Infinities and NaN in the others become zeros too, and the unit is marked: its rows add those that they
//     see at the end. Tiles seen in whole need neither.
#pragma once
#include "prompt.cu"

struct pt_info { int base, len, tok0, head, lo, nsink, n0, n1, sk, end, dirty; };

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint64_t *bar)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 :: "r"(irx_smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
                    "r"(irx_smem_u32(bar)) : "memory");
}

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float pt_max3(float a, float b, float c)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// First token of key tile j, and whether some row of tokens [first, last] does not see all of it.
__device__ __forceinline__ int pt_key(const pt_info &f, int j) { return j < f.nsink ? 128 * j : f.lo + 128 * (j - f.nsink); }

// Whether the unit needs only the first 64 keys of tile j: the sinks' or the last one, when that is all there is. Not for
// head sizes up to 64, whose softmax bounds them: a second form of its step in the loop costs the first more than
// it saves (window with sinks 365 us with it, 352 without).
template <int DP>
__device__ __forceinline__ bool pt_narrow(const pt_info &f, int j) { return DP != 64 && (j < f.nsink ? f.sk : f.end) - pt_key(f, j) <= 64; }

__device__ __forceinline__ bool pt_cut(const irx_kprm_t &p, const pt_info &f, int j, int first, int last)
{
    const int kb = pt_key(f, j);
    return j < f.nsink || kb + 127 > first || (p.window && kb <= last - p.window);
}

// The lowest n bits, n any number.
__device__ __forceinline__ uint32_t pt_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

#define PT_HALF 16384                       // 128 rows of 64 columns

// All 64 f32 columns of this thread's TMEM lane, with the wait in the same statement.
__device__ __forceinline__ void pt_ld64(uint32_t taddr, float (&v)[64])
{
    uint32_t r[64];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
                 "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
                 "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                   "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                   "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                   "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr) : "memory");
#pragma unroll
    for (int i = 0; i < 64; i++) v[i] = __uint_as_float(r[i]);
}

// 32 packed columns (64 bf16 of P) into this thread's TMEM lane, then wait for the stores.
__device__ __forceinline__ void pt_st32(uint32_t taddr, const uint32_t (&v)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
                 "%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
                 "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};\n\t"
                 "tcgen05.wait::st.sync.aligned;"
                 :: "r"(taddr),
                    "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
                    "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
                    "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
                    "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}

// Two bf16 numbers less 2^-126 each.
__device__ __forceinline__ uint32_t pt_less(uint32_t x)
{
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x00800080u));
    return d;
}

// at_softmax_row (attn.cu) for W scores: P = 2^(s * sl2 - m) as bf16 pairs, and their sum.
//
// Weights are rounded to bf16, the product's type; the row's sum is of the weights as they were. The output is then 0.0018 to
// 0.0022 off the definition (norms), where its own rounding makes 0.0016. Weights as two bf16 numbers and two products, as the
// decode kernel has, for which they are no work, bring that to 0.0016 but cost a third to four fifths here: 16001 tokens 3310 us
// against 2115, a ragged batch 415 against 232, a window with sinks 470 against 358, 37 tokens 10.2 against 8.0 (the second
// halves in the scores' other columns).
//
// What differs from at_softmax_row: the FMA pipe's pairs, which end at 2^-126, lose that much once rounded, so that a weight
// below it is 0 on either pipe and adds nothing, however large its value. (From 2^-116 on that is less than half a step of a
// bf16 weight: those are the same bits.)
template <int W>
__device__ __forceinline__ float pt_weights(const float (&v)[W], float sl2, float m, uint32_t (&pk)[W / 2])
{
    float2 sa = make_float2(0.0f, 0.0f), sb = make_float2(0.0f, 0.0f);
    const float2 s2 = make_float2(sl2, sl2), nm = make_float2(-m, -m);
    const float ks = sl2 * (1.0f / 253.0f), kc = (126.0f - m) * (1.0f / 253.0f);
    const float2 k253 = make_float2(253.0f, 253.0f), kmg = make_float2(12582912.0f - 126.0f, 12582912.0f - 126.0f);
#pragma unroll
    for (int i = 0; i < W / 2; i++) {
        if ((i & 3) != 3) {
            const float2 x = __ffma2_rn(make_float2(v[2 * i], v[2 * i + 1]), s2, nm);
            const float p0 = at_ex2(x.x), p1 = at_ex2(x.y);
            pk[i] = at_pack_bf16(p0, p1);
            sa = __fadd2_rn(sa, make_float2(p0, p1));
        } else {
            const float2 y = make_float2(at_ffma_sat(v[2 * i], ks, kc), at_ffma_sat(v[2 * i + 1], ks, kc));
            const float2 t = __ffma2_rn(y, k253, kmg);
            const float2 nn = __fadd2_rn(kmg, make_float2(-t.x, -t.y));
            const float2 f = __ffma2_rn(y, k253, nn);
            float2 q = __ffma2_rn(make_float2(0.055171319384097875f, 0.055171319384097875f), f,
                                  make_float2(0.2426105373823389f, 0.2426105373823389f));
            q = __ffma2_rn(q, f, make_float2(0.6932609854947172f, 0.6932609854947172f));
            q = __ffma2_rn(q, f, make_float2(0.9999281096694117f, 0.9999281096694117f));
            const uint32_t r0 = __float_as_uint(q.x) + (__float_as_uint(t.x) << 23);
            const uint32_t r1 = __float_as_uint(q.y) + (__float_as_uint(t.y) << 23);
            pk[i] = pt_less(__byte_perm(r0 + 0x8000u, r1 + 0x8000u, 0x7632));
            sb = __fadd2_rn(sb, make_float2(__uint_as_float(r0), __uint_as_float(r1)));
        }
    }
    return (sa.x + sa.y) + (sb.x + sb.y);
}

// One softmax step of a row over W scores: masked, exponentials 2^(x - m) over the scores' columns, and into m and l. m is set
// PT_LAG above a maximum and moves when one passes it (attn.cu's lag of a factor of 256, from above: no weight is over 1, and O
// stays within the values' sum). Each row decides for itself, so that its bits do not depend on the others of its warp. before(): waits
// until O is this warp's to rescale.
#define PT_LAG 8.0f
struct pt_row {
    uint32_t tS, tO;
    int up, low, sink;                          // the columns seen: up to `up`, and from `low` on or before `sink`
    bool cut, other, first;                     // other: a scale that is not above 0
    float scale2, sl2;                          // sl2: above 0, since hidden scores are -infinity times it
};
__device__ __forceinline__ float pt_sl2(float scale2) { return scale2 == 0.0f ? 1.0f : fabsf(scale2); }

template <int DP, int W, class F>
__device__ __forceinline__ void pt_step(const pt_row &r, float &m, float &l, F before)
{
    float v[W];
    if constexpr (W == 128) tmem_ld128(r.tS, v);
    else pt_ld64(r.tS, v);
    if (r.other) {                                // the rest of the scale: a sign, or 0
        const float by = r.scale2 < 0.0f ? -1.0f : 0.0f;
#pragma unroll
        for (int c = 0; c < W; c++) v[c] *= by;
    }
    if (r.cut) {
#pragma unroll
        for (int k = 0; k < W / 32; k++) {
            const uint32_t see = pt_below(r.up + 1 - 32 * k) & (~pt_below(r.low - 32 * k) | pt_below(r.sink - 32 * k));
#pragma unroll
            for (int c = 0; c < 32; c++)
                if (!(see & (1u << c))) v[k * 32 + c] = -INFINITY;
        }
    }
    float mk[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        mk[k] = pt_max3(v[k * (W / 4)], v[k * (W / 4) + 1], v[k * (W / 4) + 2]);
#pragma unroll
        for (int c = 3; c < W / 4 - 1; c += 2) mk[k] = pt_max3(mk[k], v[k * (W / 4) + c], v[k * (W / 4) + c + 1]);
    }
    mk[0] = pt_max3(mk[0], v[W / 4 - 1], v[W / 2 - 1]);
    mk[1] = pt_max3(mk[1], v[3 * W / 4 - 1], v[W - 1]);
    float top = pt_max3(-3.0e38f, pt_max3(mk[0], mk[1], mk[2]) * r.sl2, mk[3] * r.sl2);
    top = top < INFINITY ? top : NAN;            // a score that is NaN or infinite: the row is NaN
    const bool grown = !(top <= m);
    if (r.first) {
        m = top + PT_LAG;
    } else if (__any_sync(0xffffffffu, grown)) {
        if (!before()) return;
        const float alpha = grown ? at_ex2(m - (top + PT_LAG)) : 1.0f;
        if (grown) m = top + PT_LAG;
        l *= alpha;
#pragma unroll 1
        for (int cc = 0; cc < DP / 32; cc++) {
            float o[32];
            tmem_ld32(r.tO + cc * 32, o);
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] *= alpha;
            tmem_st32(r.tO + cc * 32, o);
        }
    }
    uint32_t pk[W / 2];
    if (r.cut) {                                  // all on the MUFU, whose weight of a hidden key, 2^-infinity, is exactly 0
        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < W / 2; i++) {
            const float2 x = __ffma2_rn(make_float2(v[2 * i], v[2 * i + 1]), make_float2(r.sl2, r.sl2), make_float2(-m, -m));
            const float p0 = at_ex2(x.x), p1 = at_ex2(x.y);
            pk[i] = at_pack_bf16(p0, p1);
            sum = __fadd2_rn(sum, make_float2(p0, p1));
        }
        l += sum.x + sum.y;
    } else {
        l += pt_weights<W>(v, r.sl2, m, pk);
    }
    if constexpr (W == 128) tmem_st64(r.tS, pk);
    else pt_st32(r.tS, pk);
}

template <int DP>
__device__ __forceinline__ void pt_body(const irx_kprm_t &p)
{
    constexpr int NB = DP / 64, TILE = NB * PT_HALF;
    irx_pdl_enter();
    extern __shared__ __align__(1024) unsigned char pt_smem[];
    unsigned char *sq = pt_smem, *sk = sq + 2 * TILE, *sv = sk + 2 * TILE;
    if (irx_smem_u32(pt_smem) & 1023u) {
        if (threadIdx.x == 0) atomicOr(p.err, IRX_KERR_TIMEOUT);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(sv + 2 * TILE);
    uint64_t *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7;
    uint64_t *s_full = bars + 9, *p_full = bars + 11, *pv_done = bars + 13, *done = bars + 15, *q_empty = bars + 16, *o_free = bars + 17;
    uint64_t *u_full = bars + 19, *u_empty = bars + 21, *v_ok = bars + 23;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(bars + 25);
    volatile pt_info *infos = reinterpret_cast<volatile pt_info *>(bars + 26);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = p.group, tp = 128 / g;
    if (threadIdx.x < 25) {
        const int i = threadIdx.x;          // p_full, o_free: a tile's rows; u_empty: MMA, 8 softmax and 2 value warps
        irx_mbar_init(&bars[i], i == 11 || i == 12 || i == 17 || i == 18 ? 128 : i == 21 || i == 22 ? 11 : i >= 23 ? 2 : 1);
        irx_fence_mbar_init();
        if (i == 0) {
            tma_prefetch_desc(&p.tma_q);
            tma_prefetch_desc(&p.tma_k);
            tma_prefetch_desc(&p.tma_v);
        }
    }
    if (warp == 9) tmem_alloc(tslot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = *tslot;
    auto read = [&](int us) {
        pt_info f;
        f.base = infos[us].base; f.len = infos[us].len; f.tok0 = infos[us].tok0; f.head = infos[us].head;
        f.lo = infos[us].lo; f.nsink = infos[us].nsink; f.n0 = infos[us].n0; f.n1 = infos[us].n1; f.sk = infos[us].sk;
        f.end = infos[us].end; f.dirty = 0;
        return f;
    };
    if (warp >= 8) {
      at_reg_dec();
      if (warp == 8) {                                        // units and loads
        int kv = 0;
        const pr_list list = pr_start(p, pr_rows{1, 2 * tp});
        int ok = 1;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            const int64_t u = pr_turn(uc);
            pt_info f = {};
            if (u < list.units) {
                const pr_unit un = pr_find(p, list, u);
                f.base = un.base; f.len = un.len; f.head = un.head;
                f.tok0 = un.tile * 2 * tp;
                const int e0 = min(f.tok0 + tp, f.len), e1 = min(f.tok0 + 2 * tp, f.len);
                f.end = e1;
                f.lo = p.window ? max(0, f.tok0 - p.window + 1) : 0;
                f.sk = min(p.sinks, f.lo);
                f.nsink = (f.sk + 127) / 128;
                f.n0 = f.nsink + (e0 - f.lo + 127) / 128;
                f.n1 = e1 > e0 ? f.nsink + (e1 - f.lo + 127) / 128 : 0;
            }
            if (lane == 0) {
                ok = at_wait(&u_empty[us], ((uc >> 1) & 1) ^ 1, p.err);
                if (ok) {
                    infos[us].base = f.base; infos[us].len = f.len; infos[us].tok0 = f.tok0; infos[us].head = f.head;
                    infos[us].lo = f.lo; infos[us].nsink = f.nsink; infos[us].n0 = f.n0; infos[us].n1 = f.n1;
                    infos[us].sk = f.sk; infos[us].end = f.end; infos[us].dirty = 0;
                    irx_mbar_arrive(&u_full[us]);
                }
                if (ok && f.n0) {
                    const int nmax = max(f.n0, f.n1), nt = f.n1 ? 2 : 1;
                    if (uc > 0) ok = at_wait(q_empty, (uc - 1) & 1, p.err);
                    if (ok) {
                        irx_mbar_expect_tx(q_full, (uint32_t)(nt * NB * tp * g * 128));
                        for (int t = 0; t < nt; t++)
                            for (int b = 0; b < NB; b++)
                                tma_load_4d(sq + t * TILE + b * PT_HALF, &p.tma_q, 64 * b, 0, f.head, f.base + f.tok0 + t * tp, q_full);
                    }
                    for (int t = 0; t <= nmax && ok; t++) {
                        if (t < nmax) {
                            const int gi = kv + t, sl = gi & 1;
                            if (!(ok = at_wait(&k_empty[sl], ((gi >> 1) & 1) ^ 1, p.err))) break;
                            irx_mbar_expect_tx(&k_full[sl], TILE);
                            for (int b = 0; b < NB; b++)
                                tma_load_3d(sk + sl * TILE + b * PT_HALF, &p.tma_k, 64 * b, f.head, f.base + pt_key(f, t), &k_full[sl]);
                        }
                        if (t >= 1) {
                            const int gi = kv + t - 1, sl = gi & 1;
                            if (!(ok = at_wait(&v_empty[sl], ((gi >> 1) & 1) ^ 1, p.err))) break;
                            irx_mbar_expect_tx(&v_full[sl], TILE);
                            for (int b = 0; b < NB; b++)
                                tma_load_3d(sv + sl * TILE + b * PT_HALF, &p.tma_v, 64 * b, f.head, f.base + pt_key(f, t - 1), &v_full[sl]);
                        }
                    }
                    kv += nmax;
                }
                if (!f.n0) ok = 0;                            // that was the end
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
        }
      } else if (warp == 9) {
        if (elect_one()) {                                    // MMA: P0 V, S0', P1 V, S1' per key tile
            const uint32_t id_qk = umma_idesc_bf16(128, 128, 0), id_qk64 = umma_idesc_bf16(128, 64, 0), id_pv = umma_idesc_bf16(128, DP, 1);
            const uint32_t sq_a = irx_smem_u32(sq), sk_a = irx_smem_u32(sk), sv_a = irx_smem_u32(sv);
            bool ok = true;
            int kv = 0, it0 = 0, it1 = 0, uo0 = 0, uo1 = 0;
            for (int uc = 0; ok; uc++) {
                const int us = uc & 1;
                if (!(ok = at_wait(&u_full[us], (uc >> 1) & 1, p.err))) break;
                const pt_info f = read(us);
                const int n0 = f.n0, n1 = f.n1, nmax = max(n0, n1);
                irx_mbar_arrive(&u_empty[us]);
                if (!n0) break;
                int sleft = n0 + n1;                          // score products of this unit still to issue
                if (!(ok = at_wait(q_full, uc & 1, p.err))) break;
                for (int j = -1; j < nmax && ok; j++) {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        const int nt = t ? n1 : n0;
                        if (!ok) break;
                        if (j >= 0 && j < nt) {               // O_t (+)= P_t V_j
                            const int gi = kv + j;
                            if (j == 0 && (t ? uo1 : uo0) > 0 && !(ok = at_wait(&o_free[t], ((t ? uo1 : uo0) - 1) & 1, p.err))) break;
                            if (!(ok = at_wait(&p_full[t], ((t ? it1 : it0) + j) & 1, p.err))) break;
                            if (!(ok = at_wait(&v_full[gi & 1], (gi >> 1) & 1, p.err))) break;
                            if (!(ok = at_wait(&v_ok[gi & 1], (gi >> 1) & 1, p.err))) break;
                            tc_fence_after();
                            const uint32_t bv = sv_a + (gi & 1) * TILE;
                            const bool narrow = pt_narrow<DP>(f, j);
#pragma unroll
                            for (int kk = 0; kk < 8; kk++)
                                if (kk < 4 || !narrow)
                                    umma_bf16_tmem_a(tbase + 256 + t * 128, tbase + t * 128 + kk * 8,
                                                     umma_desc_sw128(bv + kk * 16 * 128, PT_HALF, 1024), id_pv, (j | kk) != 0);
                            umma_commit(&pv_done[t]);
                        }
                        if (j + 1 < nt) {                     // S_t = Q_t K_{j+1}^T
                            const int gi = kv + j + 1;
                            if (!(ok = at_wait(&k_full[gi & 1], (gi >> 1) & 1, p.err))) break;
                            tc_fence_after();
                            const uint32_t aq = sq_a + t * TILE, bk = sk_a + (gi & 1) * TILE, id = pt_narrow<DP>(f, j + 1) ? id_qk64 : id_qk;
#pragma unroll
                            for (int kk = 0; kk < DP / 16; kk++)
                                umma_bf16(tbase + t * 128, at_kmajor_desc(aq, kk), at_kmajor_desc(bk, kk), id, kk > 0);
                            umma_commit(&s_full[t]);
                            if (--sleft == 0) umma_commit(q_empty);
                        }
                    }
                    if (!ok) break;
                    if (j >= 0) umma_commit(&v_empty[(kv + j) & 1]);
                    if (j + 1 < nmax) umma_commit(&k_empty[(kv + j + 1) & 1]);
                }
                if (!ok) break;
                it0 += n0;
                uo0++;
                if (n1) { it1 += n1; uo1++; }
                kv += nmax;
            }
            umma_commit(done);
            at_wait(done, 0, p.err);
        }
        __syncwarp();
        asm volatile("bar.sync 1, 288;" ::: "memory");         // the softmax warps are done with TMEM
        tc_fence_after();
        tmem_dealloc(tbase, 512);
      } else {                                                // warps 10 and 11: 64 rows each of every value tile
        int ok = 1, kv = 0;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            ok = __all_sync(0xffffffffu, at_wait(&u_full[us], (uc >> 1) & 1, p.err));
            if (!ok) break;
            const pt_info f = read(us);
            if (!f.n0) break;
            const int nmax = max(f.n0, f.n1);
            for (int j = 0; j < nmax; j++) {
                const int gi = kv + j;
                ok = __all_sync(0xffffffffu, at_wait(&v_full[gi & 1], (gi >> 1) & 1, p.err));
                if (!ok) break;
                if (pt_cut(p, f, j, f.tok0, f.end - 1)) {
                    const int seen = (j < f.nsink ? f.sk : f.end) - pt_key(f, j);
                    uint4 *v = reinterpret_cast<uint4 *>(sv + (gi & 1) * TILE);
                    const int quads = pt_narrow<DP>(f, j) ? 8 : 16;       // rows are looked at in fours: half of them by each warp
                    uint32_t worst = 0;                       // the largest magnitudes of either half, as integers
#pragma unroll 4
                    for (int i = 0; i < NB * quads; i++) {
                        const int blk = i >= quads, row = ((warp - 10) * quads + i - blk * quads) * 4 + (lane >> 3);
                        uint4 *at = v + blk * (PT_HALF / 16) + row * 8 + (lane & 7);
                        const uint4 x = *at;
                        if (row >= seen) *at = make_uint4(0u, 0u, 0u, 0u);
                        else worst = __vmaxu2(__vmaxu2(worst, __vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu)),
                                              __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu));
                    }
                    // an exponent of all ones: find them
                    const bool odd = __any_sync(0xffffffffu, (worst & 0xffffu) >= 0x7f80u || worst >> 16 >= 0x7f80u);
                    if (odd)
                        for (int i = 0; i < NB * quads; i++) {
                            const int blk = i >= quads, row = ((warp - 10) * quads + i - blk * quads) * 4 + (lane >> 3);
                            uint4 *at = v + blk * (PT_HALF / 16) + row * 8 + (lane & 7);
                            const uint4 x = *at;
                            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int e = 0; e < 4; e++) w[e] &= ~__vcmpeq2(w[e] & 0x7f807f80u, 0x7f807f80u);
                            *at = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    if (odd) infos[us].dirty = 1;
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) irx_mbar_arrive(&v_ok[gi & 1]);
            }
            kv += nmax;
            if (lane == 0) irx_mbar_arrive(&u_empty[us]);
        }
      }
    } else {                                                   // softmax: warps 0-3 tile 0, 4-7 tile 1
        at_reg_inc();
        const int t = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t tl = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tbase + tl + t * 128, tO = tbase + tl + 256 + t * 128;
        const float sl2 = pt_sl2(p.scale2);
        uint4 *stage = reinterpret_cast<uint4 *>(sv + 2 * TILE + 1024) + warp * 256;
        const int inv_g = (65535 + g) / g, tok_stride = p.heads * p.d;        // row / g = (row * inv_g) >> 16 below 128
        const int mytok = t * tp + r / g, myhead = r % g;      // within the unit, within the group
        bool ok = true;
        int it = 0;
        for (int uc = 0; ok; uc++) {
            const int us = uc & 1;
            ok = __all_sync(0xffffffffu, at_wait(&u_full[us], (uc >> 1) & 1, p.err));
            if (!ok) break;
            const pt_info f = read(us);
            if (!f.n0) break;
            const int n = t ? f.n1 : f.n0;
            const int tok = f.tok0 + mytok;
            const int first = f.tok0 + t * tp, last = min(first + tp, f.len) - 1;
            float m = -3.0e38f, l = 0.0f;
            for (int j = 0; j < n; j++) {
                ok = __all_sync(0xffffffffu, at_wait(&s_full[t], (it + j) & 1, p.err));
                if (!ok) break;
                tc_fence_after();
                const int kb = pt_key(f, j);
                const bool edge = j >= f.nsink && p.window && kb <= last - p.window;
                const int up = (j < f.nsink ? min(tok, f.sk - 1) : tok) - kb, low = edge ? tok - p.window + 1 - kb : -0x40000000;
                auto done_before = [&]() {                    // the product of the step before, which writes O
                    ok = __all_sync(0xffffffffu, at_wait(&pv_done[t], (it + j - 1) & 1, p.err));
                    tc_fence_after();
                    return ok;
                };
                const pt_row row = {tS, tO, up, low, p.sinks - kb, edge || j < f.nsink || kb + 127 > first, !(p.scale2 > 0.0f), j == 0, p.scale2, sl2};
                if (pt_narrow<DP>(f, j)) pt_step<DP, 64>(row, m, l, done_before);
                else pt_step<DP, 128>(row, m, l, done_before);
                if (!ok) break;
                tc_fence_before();
                irx_mbar_arrive(&p_full[t]);
            }
            if (!ok) break;
            it += n;
            if (n) {
                ok = __all_sync(0xffffffffu, at_wait(&pv_done[t], (it - 1) & 1, p.err));
                if (!ok) break;
                tc_fence_after();
                const bool mine = r < tp * g && tok < f.len;
                const bool odd = infos[us].dirty != 0;
                const float inv = m > -2.9e38f ? 1.0f / l : NAN;      // (every score -infinity, or NaN: NaN)
                const int64_t orow = (int64_t)(f.base + tok) * p.heads + f.head * g + myhead;
                if (mine && p.lse) p.lse[orow] = m < -2.9e38f ? -INFINITY : (m + log2f(l)) * 0.6931471806f;
                __nv_bfloat16 *o_at = reinterpret_cast<__nv_bfloat16 *>(p.o) + ((int64_t)(f.base + first) * p.heads + f.head * g) * p.d;
                const int rows = (last + 1 - first) * g;      // of this tile
#pragma unroll 1
                for (int cc = 0; cc < DP / 32; cc++) {
                    float o[32];
                    tmem_ld32(tO + cc * 32, o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] *= inv;
                    if (odd && mine) {                        // the infinities and NaN this row sees in the cut tiles
                        for (int j = 0; j < n; j++) {
                            if (!pt_cut(p, f, j, f.tok0, f.end - 1)) continue;
                            const int kb = pt_key(f, j), ke = min(kb + 128, j < f.nsink ? f.sk : tok + 1);
                            for (int key = kb; key < ke; key++) {
                                if (p.window && key <= tok - p.window && key >= p.sinks) continue;
                                const __nv_bfloat16 *vr = reinterpret_cast<const __nv_bfloat16 *>(p.v) + (int64_t)(f.base + key) * p.kv_stride +
                                                          (int64_t)f.head * p.d + cc * 32;
#pragma unroll
                                for (int e = 0; e < 32; e++) {
                                    const float x = cc * 32 + e < p.d ? __bfloat162float(vr[e]) : 0.0f;
                                    if (!(fabsf(x) < INFINITY)) o[e] += x;
                                }
                            }
                        }
                    }
                    // 64 columns at a time through the warp's 4 KB, so that a store covers four rows' 128 bytes, not 32 rows'
                    // 16 (chunks of 16 bytes, swizzled by row)
                    uint4 *st = stage + lane * 8;
#pragma unroll
                    for (int j8 = 0; j8 < 4; j8++)
                        st[((cc & 1) * 4 + j8) ^ (lane & 7)] = make_uint4(at_pack_bf16(o[j8 * 8 + 0], o[j8 * 8 + 1]), at_pack_bf16(o[j8 * 8 + 2], o[j8 * 8 + 3]),
                                                                          at_pack_bf16(o[j8 * 8 + 4], o[j8 * 8 + 5]), at_pack_bf16(o[j8 * 8 + 6], o[j8 * 8 + 7]));
                    if (!(cc & 1)) continue;
                    __syncwarp();
                    const int col = (cc >> 1) * 64 + (lane & 7) * 8;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int row = i * 4 + (lane >> 3), full = (warp & 3) * 32 + row, tk = (full * inv_g) >> 16;
                        if (full < rows && col < p.d)
                            *reinterpret_cast<uint4 *>(o_at + tk * tok_stride + (full - tk * g) * p.d + col) = stage[row * 8 + ((lane & 7) ^ (row & 7))];
                    }
                    __syncwarp();
                }
                tc_fence_before();
                irx_mbar_arrive(&o_free[t]);
            }
            __syncwarp();
            if (lane == 0) irx_mbar_arrive(&u_empty[us]);
        }
        tc_fence_before();
        asm volatile("bar.arrive 1, 288;" ::: "memory");
    }
}

extern "C" __global__ void __launch_bounds__(AT_THREADS, 1) irx_prompt_tc_64(const __grid_constant__ irx_kprm_t p) { pt_body<64>(p); }
extern "C" __global__ void __launch_bounds__(AT_THREADS, 1) irx_prompt_tc_128(const __grid_constant__ irx_kprm_t p) { pt_body<128>(p); }
