// The shared prefix on tcgen05 / TMEM: the rows that all sequences have on a key head against the prefix's keys and values.
//
// One CTA = one key head, one slice of the prefix and two tiles of 128 rows (PAIR), or one tile where a key head has no more rows.
// K / V tiles of 128 positions by TMA straight from the prefix's ring, zeros past its end. Two groups of four softmax warps:
// of a PAIR each has a row tile, and the two share every K / V tile (a CTA with one row tile would need 64 KB of L2 for 32 KB
// worth of work: 119 bytes a cycle and SM, where L2 gives about 64); of a single tile each has every other K / V tile, with an S, an O,
// maxima and sums of its own, and the halves are added at the end.
//
//   S = Q K^T       tcgen05.mma into TMEM
//   P               one thread per row: maximum, 2^(s - m) written over S as matrix operand: fp16, or bf16 as hi + lo pairs (bf16's 8 bits
//                   are fewer than a result of that type has)
//   O += P V        tcgen05.mma with P as the A operand from TMEM, V as it lies in memory (MN-major B operand)
// The reference of a row's weights is one of an earlier tile while that serves: O is rescaled only where a tile's maximum is well above it. The
// maximum comes first all the same. (Half of the weights by the old reference while the maximum is found, and again where it turned out too low:
// 183 us against 178 for 64 x 8 tokens behind 16384 positions, 94 against 93 for 64 behind 32768 in bf16.)
//
// Rows of a tile: p_tokens tokens of rep heads, heads fastest (a three-dimensional TMA box over [head_dim][heads][tokens]). Where rep does
// not divide 128 the last rows of a tile are left over: what lies in their shared memory never reaches another row.
//
//   warp 0     TMA: Q once, K and V tiles in stages
//   warp 1     one lane issues tcgen05.mma / tcgen05.commit
//   warp 2     owns the TMEM allocation (512 columns)
//   warps 4-11 softmax and output
// Every mbarrier wait is bounded; on a timeout the CTA raises the status word and winds down.
#include <cuda.h>
#include "engine.h"
#include "launchers_batch.h"
#include "sm100_attn.cuh"

namespace gehtp {

using namespace sm100;

// what a wait that ran out leaves for gehtp_attn_shared_status
__device__ unsigned int g_shared_status;

namespace {

constexpr uint32_t BKV = 128;
constexpr int NTHREADS = 384;
// A row's weights are 2^(s - reference + kLow), the reference a maximum of an earlier tile. It is made again, O with it, where a tile would have a weight
// above 2^kMost. fp16 ends at 2^16 and has 11 bits down to 2^-14: 2^-26 of the row's largest weight, and parts of them down to
// 2^-37. With references at the maximum itself, weights below 2^-25 were gone from O though not from the sum. bf16 has fp32's range.
template <bool BF> constexpr float kLow = BF ? 0.0f : 12.0f;
template <bool BF> constexpr float kMost = BF ? 14.0f : 15.5f;

// stages of K and of V tiles: as many as 227 KB hold behind the rows' tiles
template <int DB, bool PAIR>
__host__ __device__ constexpr int kv_stages() { return DB == 2 ? (PAIR ? 2 : 3) : 4; }

// whether the phase is complete, without waiting
__device__ __forceinline__ uint32_t mbar_seen(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    return ok;
}

template <int ST>
struct __align__(8) PBars {
    uint64_t q_full, kv_full[ST], kv_empty[ST], s_full[2], p_full[2], o_full, merge, drained;
    uint32_t tmem_base, abort_flag;
};

// V boxes of 128 positions x 64 values: 8-position groups 1024 bytes apart, the second 64 values 16384 bytes further
__device__ __forceinline__ uint64_t desc_v128(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(16384 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// 2^(s sc + off) of 32 scores as 16 words of fp16 pairs; adds the values to l
__device__ __forceinline__ void probs32_h(const uint32_t (&v)[32], uint32_t (&w)[32], float sc, float off, float2 (&l)[2]) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float2 x = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), make_float2(sc, sc), make_float2(off, off));
        const float2 e = make_float2(ex2(x.x), ex2(x.y));
        l[i & 1] = add2(l[i & 1], e);
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(e.y), "f"(e.x));
    }
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// largest of a row's 128 scores
__device__ __forceinline__ float max128(const uint32_t (&v)[4][32]) {
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < 4; c++)
#pragma unroll
        for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1]));
    return max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
        ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr) : "memory");
}

// 2^(s sc + off) of 32 scores as matrix operand to TMEM; adds the values to l
template <bool BF>
__device__ __forceinline__ void weights32(uint32_t taddr, const uint32_t (&v)[32], float sc, float off, float2 (&l)[2]) {
    uint32_t w[32];
    if (BF) {
        probs32<false>(v, w, sc, off, 0u, l);
        tmem_st32(taddr, w);
    } else {
        probs32_h(v, w, sc, off, l);
        tmem_st16(taddr, w);
    }
}

// BF: bf16. DB: head_dim in units of 64
template <bool BF, int DB, bool PAIR>
__global__ void __launch_bounds__(NTHREADS, 1)
shared_prefix_sm100_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv, const SharedArgs A) {
    extern __shared__ unsigned char smem_raw[];
    constexpr int ST = kv_stages<DB, PAIR>();
    constexpr uint32_t BOX = 128 * 64 * 2, TILE = DB * BOX, NQ = PAIR ? 2 : 1, FMT = BF ? IDESC_BF16 : 0u;
    unsigned char* smem = (unsigned char*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* sQ = smem;
    unsigned char* sK = sQ + NQ * TILE;
    unsigned char* sV = sK + ST * TILE;
    PBars<ST>* bars = (PBars<ST>*)(sV + ST * TILE);
    volatile uint32_t* abort_flag = &bars->abort_flag;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t h = blockIdx.y, slice = blockIdx.z, tile0 = blockIdx.x * NQ;
    const uint32_t from = slice * A.p_len, to = min(A.n_prefix, from + A.p_len), n_kt = (to - from + BKV - 1) / BKV;
    const uint32_t heads = A.kv_heads * A.rep;
    const bool two = PAIR && tile0 + 1 < A.p_tiles;               // an odd number of row tiles leaves the last CTA one
    const uint32_t box_rows = A.p_tokens * A.rep;

    if (threadIdx.x == 32)
        for (const CUtensorMap* map : {&tmap_q, &tmap_kv}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    if (threadIdx.x == 0) {
        mbar_init(&bars->q_full, 1); mbar_init(&bars->o_full, 1); mbar_init(&bars->drained, 1); mbar_init(&bars->merge, 8);
        for (int s = 0; s < ST; s++) { mbar_init(&bars->kv_full[s], 1); mbar_init(&bars->kv_empty[s], 1); }
        for (int s = 0; s < 2; s++) { mbar_init(&bars->s_full[s], 1); mbar_init(&bars->p_full[s], 4); }
        bars->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bars->tmem_base;
    pdl_wait();
    if (blockIdx.x + blockIdx.y + blockIdx.z == 0) {
        if (threadIdx.x == 0) {
            A.next[0] = A.next[1] = 0;
            asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(A.start), "l"(A.token) : "memory");
        }
        __syncthreads();
    }
    pdl_release();     // behind the wait: the tails' kernel starts beside this one, and by the token it sees all that this thread does

    if (warp < 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            mbar_expect_tx(&bars->q_full, (two ? 2 : 1) * DB * box_rows * 128);
            for (uint32_t t = 0; t < (two ? 2u : 1u); t++)
#pragma unroll
                for (uint32_t d = 0; d < DB; d++)
                    tma_load_3d(sQ + t * TILE + d * BOX, &tmap_q, (int)(d * 64), (int)(h * A.rep), (int)((tile0 + t) * A.p_tokens), &bars->q_full);
            uint32_t n = 0;
            for (uint32_t j = 0; j < n_kt && !*abort_flag; j++) {
                const uint32_t s = j % ST, ph = (j / ST) & 1;
                const int y = (int)(from + j * BKV);
                if (!mbar_wait_or_abort(&bars->kv_empty[s], ph ^ 1, abort_flag)) { *abort_flag = 1; break; }
                mbar_expect_tx(&bars->kv_full[s], 2 * TILE);
#pragma unroll
                for (uint32_t d = 0; d < DB; d++) tma_load_2d(sK + s * TILE + d * BOX, &tmap_kv, (int)((h * DB + d) * 64), y, &bars->kv_full[s]);
#pragma unroll
                for (uint32_t d = 0; d < DB; d++) tma_load_2d(sV + s * TILE + d * BOX, &tmap_kv, (int)(((A.kv_heads + h) * DB + d) * 64), y, &bars->kv_full[s]);
                n++;
            }
            if (*abort_flag) {   // copies already requested must land before the CTA may go away
                mbar_wait(&bars->q_full, 0);
                for (uint32_t j = n > ST ? n - ST : 0; j < n; j++) mbar_wait(&bars->kv_full[j % ST], (j / ST) & 1);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        // The whole warp walks the tiles, so that counters, descriptors and barrier addresses are warp-uniform values; lane 0 issues. (One
        // lane on its own took 84 cycles to an instruction that the tensor core runs in 64. A look at a complete barrier takes some
        // 230: K and V of a tile share one, and the next barrier is looked at while instructions in front of it are issued.)
        const uint64_t dq = umma_desc(smem_u32(sQ)), dk = umma_desc(smem_u32(sK)), dv = desc_v128(smem_u32(sV));
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t seen = 0) {
            if (!__all_sync(0xffffffffu, seen)) ok = __all_sync(0xffffffffu, ok && mbar_wait_or_abort(bar, parity, abort_flag));
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return ok;
        };
        auto commit = [&](uint64_t* bar) { if (lane == 0) umma_commit(bar); };
        // S of group t: row tile `q` against the K tile of stage s
        auto issue_s = [&](uint32_t t, uint32_t q, uint32_t s) {
            if (lane == 0) {
                const uint64_t a = dq + q * (TILE >> 4), b = dk + s * (TILE >> 4);
#pragma unroll
                for (uint32_t k = 0; k < DB * 4; k++)
                    umma_f16(tmem + t * 128, a + (k >> 2) * (BOX >> 4) + (k & 3) * 2, b + (k >> 2) * (BOX >> 4) + (k & 3) * 2, idesc_f16(128) | FMT, k ? 1u : 0u);
                umma_commit(&bars->s_full[t]);
            }
        };
        auto issue_o = [&](uint32_t t, uint32_t s, bool first) {
            if (lane == 0) {
                const uint64_t b = dv + s * (TILE >> 4);
#pragma unroll
                for (uint32_t k = 0; k < 8; k++)                     // 16 positions = two 8-position groups = 2048 bytes; bit 16: B is MN-major
#pragma unroll
                    for (uint32_t part = 0; part < (BF ? 2u : 1u); part++)
                        umma_f16_ta(tmem + 256 + t * 128, tmem + t * 128 + (k >> 1) * 32 + part * 16 + (k & 1) * 8, b + k * (2048 >> 4),
                                    idesc_f16(DB * 64) | FMT | (1u << 16), (part || k) ? 1u : first ? 0u : 1u);
            }
        };
        uint32_t s = 0, ph = 0, s1 = 0, ph1 = 0;                     // stage and phase of the tile whose P is next, and of the one whose S is
        auto step = [&](uint32_t& st, uint32_t& p) { if (++st == (uint32_t)ST) { st = 0; p ^= 1; } };
        wait(&bars->q_full, 0);
        if (PAIR) {
            if (wait(&bars->kv_full[0], 0)) {
                issue_s(0, 0, 0);
                if (two) issue_s(1, 1, 0);
            }
            step(s1, ph1);
            uint32_t seen0 = 0;
            for (uint32_t j = 0; ok && j < n_kt; j++) {
                const bool more = j + 1 < n_kt;
                if (!wait(&bars->p_full[0], j & 1, seen0)) break;
                const uint32_t seen_kv = mbar_seen(&bars->kv_full[s1], ph1);
                issue_o(0, s, j == 0);
                const uint32_t seen1 = two ? mbar_seen(&bars->p_full[1], j & 1) : 0;
                if (more) {
                    if (!wait(&bars->kv_full[s1], ph1, seen_kv)) break;
                    issue_s(0, 0, s1);
                }
                if (two) {
                    if (!wait(&bars->p_full[1], j & 1, seen1)) break;
                    issue_o(1, s, j == 0);
                }
                commit(&bars->kv_empty[s]);
                seen0 = mbar_seen(&bars->p_full[0], (j + 1) & 1);
                if (more && two) issue_s(1, 1, s1);
                step(s, ph);
                step(s1, ph1);
            }
        } else {
            for (uint32_t j = 0; j < 2 && j < n_kt && wait(&bars->kv_full[s1], ph1); j++) {
                issue_s(j, 0, s1);
                step(s1, ph1);
            }
            for (uint32_t j = 0; ok && j < n_kt; j++) {
                if (!wait(&bars->p_full[j & 1], (j >> 1) & 1)) break;
                issue_o(j & 1, s, j < 2);
                commit(&bars->kv_empty[s]);
                step(s, ph);
                if (j + 2 < n_kt) {                                  // over the P just read: products run in the order they are issued
                    if (!wait(&bars->kv_full[s1], ph1)) break;
                    issue_s(j & 1, 0, s1);
                    step(s1, ph1);
                }
            }
        }
        if (ok) {
            commit(&bars->o_full);
        } else {                 // products under way still read shared memory and write the TMEM that the CTA is about to give back
            if (lane == 0) *abort_flag = 1;
            commit(&bars->drained);
            mbar_wait(&bars->drained, 0);
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------ softmax and output: one thread per row and group
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");    // 256 x 200 + 128 x 104 = 384 x 168, what the CTA was launched with
        const uint32_t t = (warp - 4) >> 2, quarter = warp & 3;
        const uint32_t ts = tmem + ((quarter * 32) << 16) + t * 128, to_ = ts + 256;
        float ref = -INFINITY;                                   // score that the weights are referred to
        float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        bool ok = true;
        const bool works = t == 0 || (PAIR ? two : n_kt > 1);
        uint32_t round = 0;
#pragma unroll 1
        for (uint32_t j = PAIR ? 0 : t; works && j < n_kt; j += PAIR ? 1 : 2, round++) {
            ok = !__any_sync(0xffffffffu, *abort_flag != 0) && __all_sync(0xffffffffu, mbar_wait_or_abort(&bars->s_full[t], round & 1, abort_flag));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t v[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(ts + c * 32, v[c]);
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld_wait(v[c]);
            const int hi = (int)(A.n_prefix - 1 - (from + j * BKV));       // last column of the tile that is a position of the prefix
            if (hi < (int)BKV - 1) {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int i = 0; i < 32; i++) v[c][i] = c * 32 + i <= hi ? v[c][i] : 0xff800000u;
            }
            const float top = max128(v);
            if (round == 0) {
                ref = top;
            } else {
                // O is at rest: s_full of this tile came after the group's products of the tile before
                const bool raise = fmaf(top - ref, A.sc, kLow<BF>) > kMost<BF>;
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? ex2((ref - top) * A.sc) : 1.0f;
                    if (raise) ref = top;
#pragma unroll
                    for (int i = 0; i < 2; i++) { l2[i].x *= f; l2[i].y *= f; }
#pragma unroll 1
                    for (int c = 0; c < DB * 4; c++) {
                        uint32_t x[16];
                        tmem_ld16(to_ + c * 16, x);
                        tmem_ld_wait(x);
#pragma unroll
                        for (int i = 0; i < 16; i++) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
                        tmem_st16(to_ + c * 16, x);
                    }
                    tmem_st_wait();
                }
            }
            // The difference first: in s sc - ref sc the second product is rounded, by more than a power of two where scores are far out. (Without:
            // 178 us for 181, 64 x 8 tokens behind 16384 positions.)
            const float from = ref == -INFINITY ? 0.0f : -ref, off = ref == -INFINITY ? 0.0f : kLow<BF>;
#pragma unroll
            for (int c = 0; c < 4; c++) {
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 y = add2(make_float2(__uint_as_float(v[c][i]), __uint_as_float(v[c][i + 1])), make_float2(from, from));
                    v[c][i] = __float_as_uint(y.x); v[c][i + 1] = __float_as_uint(y.y);
                }
                weights32<BF>(ts + c * 32, v[c], A.sc, off, l2);
            }
            tmem_st_wait();
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->p_full[t]);
        }
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&bars->o_full, 0, abort_flag));      // all operands have been read
        float l = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y), f0 = 1.0f, f1 = 0.0f;
        float m = ref == -INFINITY ? -INFINITY : fmaf(ref, A.sc, -kLow<BF>);
        float2* halves = (float2*)sQ;                                     // of a single row tile: {m, l} of [group][row]
        if (!PAIR && ok) {
            halves[t * 128 + quarter * 32 + lane] = make_float2(m, l);
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->merge);
            ok = __all_sync(0xffffffffu, mbar_wait_or_abort(&bars->merge, 0, abort_flag));
            const float2 a = halves[quarter * 32 + lane], b = halves[128 + quarter * 32 + lane];
            m = fmaxf(a.x, b.x);
            // a group without a maximum has no sum either, or one that is no number and stays
            f0 = a.x == -INFINITY ? (a.y == 0.0f ? 0.0f : 1.0f) : ex2(a.x - m);
            f1 = b.x == -INFINITY ? (b.y == 0.0f ? 0.0f : 1.0f) : ex2(b.x - m);
            l = a.y * f0 + b.y * f1;
        }
        const uint32_t tile = tile0 + (PAIR ? t : 0), row0 = quarter * 32;
        if (ok && tile < A.p_tiles) {
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t rows = min(A.p_tokens, A.batch * A.q_len - tile * A.p_tokens) * A.rep;
            const size_t part = (((size_t)tile * A.kv_heads + h) * A.p_slices + slice) * box_rows;
            // The warp's 32 rows by way of shared memory, so that a request touches whole rows. Of a single tile each group takes half the columns.
            constexpr uint32_t COLS = PAIR ? DB * 64 : DB * 32, CH = COLS / 4;
            float4* stage = (float4*)sK + (warp - 4) * (32 * CH);
            const uint32_t ta = tmem + ((quarter * 32) << 16) + 256 + (PAIR ? t * 128 : t * COLS);
#pragma unroll 1
            for (uint32_t c = 0; c < COLS / 16; c++) {
                uint32_t v[16], u[16];
                tmem_ld16(ta + c * 16, v);
                if (!PAIR && n_kt > 1) tmem_ld16(ta + 128 + c * 16, u);
                tmem_ld_wait(v);
                if (!PAIR && n_kt > 1) tmem_ld_wait(u);
                float x[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    x[i] = __uint_as_float(v[i]);
                    if (!PAIR) x[i] = n_kt > 1 ? fmaf(__uint_as_float(u[i]), f1, x[i] * f0) : x[i] * f0;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) stage[lane * CH + ((c * 4 + i) ^ (lane & 7))] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
            __syncwarp();
#pragma unroll 4
            for (uint32_t i = lane; i < 32 * CH; i += 32) {
                const uint32_t r = i / CH, p = i % CH;
                if (row0 + r < rows) ((float4*)(A.part_o + (part + row0 + r) * (DB * 64) + (PAIR ? 0 : t * COLS)))[p] = stage[r * CH + (p ^ (r & 7))];
            }
            if ((PAIR || t == 0) && row0 + lane < rows) A.part_ml[part + row0 + lane] = make_float2(m, l);
        }
        if (!ok) *abort_flag = 1;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 2) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        if (lane == 0 && *abort_flag) raise_status(&g_shared_status, kStatusAttnTimeout);
    }
}

template <bool BF, int DB, bool PAIR>
bool launch(cudaStream_t st, const SharedArgs& a) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    const CUtensorMapDataType type = BF ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t hd = DB * 64, heads = (cuuint64_t)a.kv_heads * a.rep, tokens = (cuuint64_t)a.batch * a.q_len;
    CUtensorMap tq, tkv;
    cuuint64_t qd[3] = {hd, heads, tokens}, qs[2] = {hd * 2, a.q_stride * 2}, kd[2] = {2 * a.kv_heads * hd, a.n_prefix}, ks[1] = {4 * a.kv_heads * hd};
    cuuint32_t qb[3] = {64, a.rep, a.p_tokens}, kb[2] = {64, BKV}, one[3] = {1, 1, 1};
    if (enc(&tq, type, 3, (void*)a.q, qd, qs, qb, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
        enc(&tkv, type, 2, (void*)a.prefix, kd, ks, kb, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    constexpr int ST = kv_stages<DB, PAIR>();
    const size_t smem = 1024 + (size_t)((PAIR ? 2 : 1) + 2 * ST) * DB * 16384 + sizeof(PBars<ST>);
    static int have[64] = {};
    if (!ensure_dyn_smem(shared_prefix_sm100_kernel<BF, DB, PAIR>, smem, have)) return false;
    const dim3 grid(PAIR ? (a.p_tiles + 1) / 2 : a.p_tiles, a.kv_heads, a.p_slices);
    g_launches++;
    return launch_pdl(shared_prefix_sm100_kernel<BF, DB, PAIR>, grid, dim3(NTHREADS), smem, st, tq, tkv, a) == cudaSuccess;
}
template <bool BF, int DB>
bool launch_pair(cudaStream_t st, const SharedArgs& a) { return a.p_tiles > 1 ? launch<BF, DB, true>(st, a) : launch<BF, DB, false>(st, a); }

}  // namespace

bool k_shared_prefix_sm100(cudaStream_t st, const SharedArgs& a, uint32_t hd, bool bf16) {
    if (hd == 128) return bf16 ? launch_pair<true, 2>(st, a) : launch_pair<false, 2>(st, a);
    return bf16 ? launch_pair<true, 1>(st, a) : launch_pair<false, 1>(st, a);
}

}  // namespace gehtp

// 0 when no bounded wait of gehtp_attn_shared's kernels on the current device has run out since the last query, else the code it
// left (and the word is cleared)
extern "C" int gehtp_attn_shared_status(void) {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, gehtp::g_shared_status, sizeof v) != cudaSuccess) { cudaGetLastError(); return -1; }
    if (v) {
        const unsigned int zero = 0;
        cudaMemcpyToSymbol(gehtp::g_shared_status, &zero, sizeof zero);
        gehtp::g.last_error = "attn shared: a K/V tile copy or a product never arrived (bounded wait ran out); the output is incomplete";
    }
    return (int)(v & 0x7fffffffu);
}
