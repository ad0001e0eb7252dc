// Drafted tokens held against the target's probabilities, from given random numbers.
//
//   p_i = softmax(target_i / T), q_i = softmax(draft_i / T); without draft logits q_i is 1 at the drafted token
//   draft i is accepted while u_i q_i(x_i) < p_i(x_i)
//   the token behind the accepted ones: the first v whose sum of r over 0 .. v is above u_n times the sum of all r, where
//   r = max(p_i - q_i, 0) at the first place i that was not accepted (p_i where the rows are alike: a sum below 1e-12), r = p_n when all were
//   T = 0: x_i is accepted while it is the lowest place of the largest logit, and the token behind is that place
//
// verify_rows_kernel: maximum and sum of 2^(x - maximum) of pieces of the rows, one pass over the logits in fp32: what the tests of
// acceptance need. A probability is then some 2^-22 off, and so is a test's border.
// verify_choose_kernel: a cluster of eight CTAs per sequence decides how many are accepted and draws the token behind them. A draw that a
// border of two tokens is next to has to go to the right one, and the borders are as many as there are tokens: this one row is taken
// in 64 bits. Every warp has a stretch of the vocabulary; its sum says in which stretch the draw ends, and that warp walks it.
#include <cooperative_groups.h>
#include <cmath>
#include <cstdio>
#include <algorithm>
#include "engine.h"
#include "launchers_batch.h"
#include "rows_common.cuh"
#include "sm100_attn.cuh"

namespace gehtp {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t MAX_DRAFTS = 64;
constexpr int RT = 256, CT = 512, CL = 8, STRETCHES = CL * CT / 32;

struct VerifyArgs {
    const void *target, *draft;             // draft NULL: drafts without probabilities (and always with T = 0)
    const int32_t *tokens, *n_drafts;
    const float* uniforms;
    int32_t *accepted, *out;
    uint32_t batch, n, vocab, pieces, piece;        // pieces of `piece` logits to a row
    size_t t_stride, d_stride;
    double inv;                             // 1 / T
    float2* part;                           // [target rows | draft rows][pieces] {maximum, sum}; T = 0: {maximum, its place}
};

struct El32 { typedef float T; static constexpr int V = 4; static __device__ float f(float x) { return x; } };
struct ElBf { typedef uint16_t T; static constexpr int V = 8; static __device__ float f(uint16_t x) { return bf2f(x); } };
struct ElHf { typedef uint16_t T; static constexpr int V = 8; static __device__ float f(uint16_t x) { return h2f(x); } };

// V logits from place e on (a multiple of V off the row's first 16-byte boundary, or in front of it): in one load where they lie in the row
// and on a boundary; places outside the row are -inf
template <class E>
__device__ __forceinline__ void load_logits(const typename E::T* row, int64_t e, int64_t end, float (&x)[E::V]) {
    const typename E::T* p = row + e;
    if (e >= 0 && e + E::V <= end && ((uintptr_t)p & 15u) == 0) {
        const uint4 v = __ldg((const uint4*)p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (E::V == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) { x[2 * i] = E::f((typename E::T)(w[i] & 0xffffu)); x[2 * i + 1] = E::f((typename E::T)(w[i] >> 16)); }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E::V; i++) x[i] = e + i >= 0 && e + i < end ? E::f(p[i]) : -INFINITY;
    }
}
// logits between the row's start and the last 16-byte boundary at or in front of it
template <class E>
__device__ __forceinline__ int lead(const typename E::T* row) { return (int)(((uintptr_t)row & 15u) / sizeof(typename E::T)); }

__device__ __forceinline__ uint32_t drafts_of(const VerifyArgs& A, uint32_t b) {
    return A.n_drafts ? (uint32_t)min(max(A.n_drafts[b], 0), (int)A.n) : A.n;
}

// {maximum, sum} of two parts of a row; a part without a maximum keeps what its sum says (0, or no number)
__device__ __forceinline__ float2 join(float2 a, float2 b, float k) {
    const float m = fmaxf(a.x, b.x);
    return make_float2(m, (a.x == m ? a.y : a.y * sm100::ex2((a.x - m) * k)) + (b.x == m ? b.y : b.y * sm100::ex2((b.x - m) * k)));
}
// {maximum, place}: the larger, of equal ones the lower place; no number wins over all
__device__ __forceinline__ bool ahead(float a, int pa, float b, int pb) {
    const bool na = a != a, nb = b != b;
    if (na != nb) return na;
    return a > b || ((a == b || na) && pa < pb);
}

template <class E, bool GREEDY>
__global__ void __launch_bounds__(RT) verify_rows_kernel(const VerifyArgs A) {
    __shared__ float2 parts[RT / 32];
    pdl_wait();
    pdl_release();
    const uint32_t t_rows = A.batch * (A.n + 1), row = blockIdx.y + blockIdx.z * gridDim.y;
    if (row >= t_rows + (A.draft ? A.batch * A.n : 0)) return;
    const bool target = row < t_rows;
    const uint32_t r = target ? row : row - t_rows, per = target ? A.n + 1 : A.n, b = r / per, i = r % per;
    if (i >= drafts_of(A, b) + (target ? 1 : 0)) return;
    const typename E::T* p = target ? (const typename E::T*)A.target + r * A.t_stride : (const typename E::T*)A.draft + r * A.d_stride;
    const int64_t first = (int64_t)blockIdx.x * A.piece - lead<E>(p), end = blockIdx.x + 1 == A.pieces ? (int64_t)A.vocab : min((int64_t)A.vocab, first + A.piece);
    const float k = (float)(A.inv * 1.4426950408889634);
    float2 best = make_float2(-INFINITY, 0.0f);
    int place = 0x7fffffff;
    for (int64_t e = first + threadIdx.x * E::V; e < end; e += RT * E::V) {
        float x[E::V];
        load_logits<E>(p, e, end, x);
        if (GREEDY) {
#pragma unroll
            for (int j = 0; j < E::V; j++)
                if (e + j >= 0 && e + j < end && ahead(x[j], (int)(e + j), best.x, place)) { best.x = x[j]; place = (int)(e + j); }
        } else {
            float m = x[0];
#pragma unroll
            for (int j = 1; j < E::V; j++) m = fmaxf(m, x[j]);
            if (m > best.x) {
                best.y = best.x == -INFINITY ? best.y : best.y * sm100::ex2((best.x - m) * k);
                best.x = m;
            }
            const float off = best.x == -INFINITY ? 0.0f : best.x;
#pragma unroll
            for (int j = 0; j < E::V; j++) best.y += sm100::ex2((x[j] - off) * k);
        }
    }
    if (GREEDY) {
        for (int o = 16; o; o >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, best.x, o);
            const int q = __shfl_xor_sync(0xffffffffu, place, o);
            if (ahead(y, q, best.x, place)) { best.x = y; place = q; }
        }
        best.y = __int_as_float(place);
    } else {
        for (int o = 16; o; o >>= 1) {
            const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, best.x, o), __shfl_xor_sync(0xffffffffu, best.y, o));
            best = join(best, y, k);
        }
    }
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < RT / 32; w++) {
            if (GREEDY) { if (ahead(parts[w].x, __float_as_int(parts[w].y), best.x, __float_as_int(best.y))) best = parts[w]; }
            else best = join(best, parts[w], k);
        }
        A.part[(size_t)row * A.pieces + blockIdx.x] = best;
    }
}

// A row's parts together, by one warp.
template <bool GREEDY>
__device__ __forceinline__ float2 whole_row(const VerifyArgs& A, size_t row) {
    const float k = (float)(A.inv * 1.4426950408889634);
    float2 x = make_float2(-INFINITY, GREEDY ? __int_as_float(0x7fffffff) : 0.0f);
    for (uint32_t i = threadIdx.x & 31; i < A.pieces; i += 32) {
        const float2 y = __ldcg(&A.part[row * A.pieces + i]);
        if (GREEDY) { if (ahead(y.x, __float_as_int(y.y), x.x, __float_as_int(x.y))) x = y; }
        else x = join(x, y, k);
    }
    for (int o = 16; o; o >>= 1) {
        const float2 y = make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o));
        if (GREEDY) { if (ahead(y.x, __float_as_int(y.y), x.x, __float_as_int(x.y))) x = y; }
        else x = join(x, y, k);
    }
    return x;
}
__device__ __forceinline__ bool sound(float2 x) { return x.y > 0.0f && isfinite(x.y) && isfinite(x.x); }

template <class E, bool GREEDY>
__global__ void __launch_bounds__(CT) verify_choose_kernel(const VerifyArgs A) {
    __shared__ double sum_p[CT / 32], sum_q[CT / 32], sum_r[CT / 32], all[STRETCHES], s_total[2], s_goal, s_upto;
    __shared__ uint8_t pass[MAX_DRAFTS];
    __shared__ float s_max[2];
    __shared__ int s_where, s_drawn;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x / CL, rank = blockIdx.x % CL;
    pdl_wait();
    pdl_release();
    const uint32_t nd = drafts_of(A, b);
    const typename E::T *target = (const typename E::T*)A.target + (size_t)b * (A.n + 1) * A.t_stride, *draft = (const typename E::T*)A.draft + (size_t)b * A.n * A.d_stride;
    // ---- which drafts pass
    for (uint32_t i = warp; i < nd; i += CT / 32) {
        const int x = A.tokens[(size_t)b * A.n + i];
        const float2 p = whole_row<GREEDY>(A, (size_t)b * (A.n + 1) + i);
        bool ok;
        if (GREEDY) {
            ok = isfinite(p.x) && x == __float_as_int(p.y);
        } else {
            const bool in = x >= 0 && (uint32_t)x < A.vocab;
            const double l2 = A.inv * 1.4426950408889634;
            double px = 0.0, qx = 1.0;
            ok = sound(p);
            if (ok && in) px = exp2(((double)E::f(target[i * A.t_stride + x]) - p.x) * l2) / p.y;
            if (A.draft) {
                const float2 q = whole_row<false>(A, (size_t)A.batch * (A.n + 1) + (size_t)b * A.n + i);
                ok = ok && sound(q);
                qx = ok && in ? exp2(((double)E::f(draft[i * A.d_stride + x]) - q.x) * l2) / q.y : 0.0;
            }
            ok = ok && (double)A.uniforms[(size_t)b * (A.n + 1) + i] * qx < px;
        }
        if (lane == 0) pass[i] = ok;
    }
    __syncthreads();
    uint32_t a = 0;
    while (a < nd && pass[a]) a++;
    const bool rejected = a < nd;
    int32_t* out = A.out + (size_t)b * (A.n + 1);
    if (rank == 0) {
        if (threadIdx.x == 0) A.accepted[b] = (int)a;
        for (uint32_t i = threadIdx.x; i <= A.n; i += CT)
            if (i != a) out[i] = i < a ? A.tokens[(size_t)b * A.n + i] : -1;
    }
    // ---- the row behind the accepted ones
    if (GREEDY) {
        if (rank == 0 && warp == 0) {
            const float2 p = whole_row<true>(A, (size_t)b * (A.n + 1) + a);
            if (lane == 0) out[a] = isfinite(p.x) ? __float_as_int(p.y) : -1;
        }
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    const bool with_q = rejected && A.draft;
    if (warp == 0) {
        const float2 p = whole_row<false>(A, (size_t)b * (A.n + 1) + a);
        if (lane == 0) s_max[0] = sound(p) ? p.x : NAN;
    }
    if (warp == 1 && with_q) {
        const float2 q = whole_row<false>(A, (size_t)A.batch * (A.n + 1) + (size_t)b * A.n + a);
        if (lane == 0) s_max[1] = sound(q) ? q.x : NAN;
    }
    __syncthreads();
    const double mp = s_max[0], mq = with_q ? s_max[1] : NAN, l2 = A.inv * 1.4426950408889634;
    if (mp != mp) {                                           // a row without a distribution (the same for the whole cluster)
        if (rank == 0 && threadIdx.x == 0) out[a] = -1;
        return;
    }
    const bool use_q = mq == mq;                              // a draft row without one takes nothing away
    const int away = rejected && !A.draft ? A.tokens[(size_t)b * A.n + a] : -1;
    const typename E::T *p = target + a * A.t_stride, *q = use_q ? draft + a * A.d_stride : nullptr;
    const int64_t vocab = A.vocab, p_lead = lead<E>(p), vecs = (vocab + p_lead + E::V - 1) / E::V;
    const uint32_t mine = rank * (CT / 32) + warp;
    const int64_t from = vecs * mine / STRETCHES, to = vecs * (mine + 1) / STRETCHES;      // the warp's stretch
    auto chance = [](float x, double l2, double m) { return exp2(((double)x - m) * l2); };
    // p - q of two such values, both products rounded on their own: equal ones leave 0
    double sp = 1.0, sq = 1.0;
    auto excess = [&](float x, float y) { return fmax(__dmul_rn(chance(x, l2, mp), sp) - __dmul_rn(chance(y, l2, mq), sq), 0.0); };
    auto block_sums = [&](double v, double* to_smem) {
        v = warp_sum_d(v);
        if (lane == 0) to_smem[warp] = v;
    };
    double tp = 0.0, tq = 0.0;
    for (int64_t j = from + lane; j < to; j += 32) {
        const int64_t e = j * E::V - p_lead;
        float x[E::V];
        load_logits<E>(p, e, vocab, x);
#pragma unroll
        for (int i = 0; i < E::V; i++) tp += e + i == away ? 0.0 : chance(x[i], l2, mp);
        if (use_q) {
            load_logits<E>(q, e, vocab, x);
#pragma unroll
            for (int i = 0; i < E::V; i++) tq += chance(x[i], l2, mq);
        }
    }
    block_sums(tp, sum_p);
    block_sums(tq, sum_q);
    cluster.sync();
    // all stretches' sums in order; every CTA for itself
    auto gather = [&](double* of) {
        for (uint32_t i = threadIdx.x; i < STRETCHES; i += CT) all[i] = cluster.map_shared_rank(of, i / (CT / 32))[i % (CT / 32)];
        __syncthreads();
    };
    bool less = false;                                        // r = p - q
    if (use_q) {
        for (int w = 0; w < 2; w++) {
            gather(w ? sum_q : sum_p);
            if (threadIdx.x == 0) {
                double t = 0.0;
                for (int i = 0; i < STRETCHES; i++) t += all[i];
                s_total[w] = t;
            }
            __syncthreads();
        }
        sp = 1.0 / s_total[0]; sq = 1.0 / s_total[1];
        double tr = 0.0;
        for (int64_t j = from + lane; j < to; j += 32) {
            const int64_t e = j * E::V - p_lead;
            float x[E::V], y[E::V];
            load_logits<E>(p, e, vocab, x);
            load_logits<E>(q, e, vocab, y);
#pragma unroll
            for (int i = 0; i < E::V; i++) tr += excess(x[i], y[i]);
        }
        block_sums(tr, sum_r);
        cluster.sync();
        gather(sum_r);
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int i = 0; i < STRETCHES; i++) t += all[i];
            s_total[0] = t;
        }
        __syncthreads();
        less = s_total[0] > 1e-12;                            // below: what the roundings of two sums leave of equal rows
    }
    if (!less) gather(sum_p);
    // p and q alike: of p, whose sums are not normalised. The drafted token alone was possible: of p with it
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < STRETCHES; i++) t += all[i];
        const double goal = fmax((double)A.uniforms[(size_t)b * (A.n + 1) + A.n] * t, 0.0);
        double upto = 0.0, front = 0.0;
        int where = -1;
        for (int i = 0; i < STRETCHES; i++) {
            if (all[i] > 0.0) { where = i; front = upto; }    // a draw of 1 and above ends in the last stretch with any
            if (upto + all[i] > goal) break;
            upto += all[i];
        }
        s_where = t > 0.0 ? where : -1;
        s_goal = goal; s_upto = front;
    }
    __syncthreads();
    if (s_where < 0) {                                        // all of p lay on the rejected token
        if (rank == 0 && threadIdx.x == 0) out[a] = away;
    } else if ((uint32_t)s_where == mine) {
        const double goal = s_goal;
        double upto = s_upto;
        int64_t found = -1, last = -1;
        for (int64_t j0 = from; j0 < to && found < 0; j0 += 32) {
            const int64_t j = j0 + lane, e = j * E::V - p_lead;
            float x[E::V], y[E::V];
            double r[E::V], sum = 0.0;
            if (j < to) {
                load_logits<E>(p, e, vocab, x);
                if (less) load_logits<E>(q, e, vocab, y);
            }
#pragma unroll
            for (int i = 0; i < E::V; i++) {
                r[i] = j >= to || e + i == away ? 0.0 : less ? excess(x[i], y[i]) : chance(x[i], l2, mp);
                sum += r[i];
            }
            double before = sum;
            for (int o = 1; o < 32; o <<= 1) {
                const double y2 = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= (uint32_t)o) before += y2;
            }
            const double end = upto + __shfl_sync(0xffffffffu, before, 31);
            double c = upto + (before - sum);
            int64_t here = -1, some = -1;
#pragma unroll
            for (int i = 0; i < E::V; i++) {
                c += r[i];
                if (r[i] > 0.0) {
                    some = e + i;
                    if (here < 0 && c > goal) here = e + i;
                }
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, here >= 0), any = __ballot_sync(0xffffffffu, some >= 0);
            if (any) last = __shfl_sync(0xffffffffu, some, 31 - __clz(any));
            if (hit) found = __shfl_sync(0xffffffffu, here, __ffs(hit) - 1);
            upto = end;
        }
        if (lane == 0) out[a] = (int)(found >= 0 ? found : last);   // the stretch's sum was above the goal: its last possible token at the latest
    }
    cluster.sync();                                           // others may still read this CTA's sums
}

const char* verify_refuses(uint32_t batch, uint32_t n, uint32_t vocab) {
    if (!batch || batch > 4096) return "verify drafts: 1 to 4096 sequences";
    if (n > MAX_DRAFTS) return "verify drafts: up to 64 drafts";
    if (!vocab || vocab > (1u << 30)) return "verify drafts: a vocabulary of 1 to 2^30";
    return nullptr;
}

// Pieces of a row: about eight CTAs an SM over all rows, of 2048 to 16384 logits
void cut_rows(uint32_t batch, uint32_t n, uint32_t vocab, uint32_t* piece, uint32_t* pieces) {
    const size_t total = (size_t)batch * (2 * n + 1) * vocab;
    uint32_t p = 2048;
    while (p < 16384 && (size_t)p * 148 * 8 < total) p *= 2;
    while (((size_t)vocab + 7 + p - 1) / p > 65535) p *= 2;
    *piece = p;
    *pieces = (uint32_t)(((size_t)vocab + 7 + p - 1) / p);    // up to seven logits in front of the first boundary
}

template <class E, bool GREEDY>
bool launch_verify(cudaStream_t st, const VerifyArgs& a) {
    const size_t rows = (size_t)a.batch * (a.n + 1) + (a.draft ? (size_t)a.batch * a.n : 0);
    const uint32_t y = (uint32_t)std::min<size_t>(rows, 32768), z = (uint32_t)((rows + y - 1) / y);
    g_launches += 2;
    if (launch_pdl(verify_rows_kernel<E, GREEDY>, dim3(a.pieces, y, z), dim3(RT), 0, st, a) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.batch * CL); cfg.blockDim = dim3(CT); cfg.stream = st;
    return launch_pdl_cluster(verify_choose_kernel<E, GREEDY>, cfg, dim3(CL, 1, 1), a) == cudaSuccess;
}

}  // namespace

bool k_verify_drafts(cudaStream_t st, const VerifyArgs& a, uint32_t dtype, bool greedy) {
    if (dtype == GEHTP_DT_F32) return greedy ? launch_verify<El32, true>(st, a) : launch_verify<El32, false>(st, a);
    if (dtype == GEHTP_DT_BF16) return greedy ? launch_verify<ElBf, true>(st, a) : launch_verify<ElBf, false>(st, a);
    return greedy ? launch_verify<ElHf, true>(st, a) : launch_verify<ElHf, false>(st, a);
}

}  // namespace gehtp

using namespace gehtp;

extern "C" size_t gehtp_verify_drafts_workspace(uint32_t batch, uint32_t n_drafts, uint32_t vocab) {
    if (const char* why = verify_refuses(batch, n_drafts, vocab)) { g.last_error = why; return 0; }
    uint32_t piece, pieces;
    cut_rows(batch, n_drafts, vocab, &piece, &pieces);
    return ((size_t)batch * (2 * n_drafts + 1) * pieces * 8 + 255) / 256 * 256;
}

extern "C" int gehtp_verify_drafts(const void* target_dev, const void* draft_dev, const int32_t* tokens_dev, const int32_t* n_drafts_dev,
                                   const float* uniforms_dev, int32_t* accepted_dev, int32_t* out_dev, uint32_t batch, uint32_t n_drafts,
                                   uint32_t vocab, uint32_t target_stride, uint32_t draft_stride, uint32_t dtype, double temperature,
                                   void* workspace_dev, size_t workspace_bytes, void* stream) {
    auto fail = [](const char* m) { g.last_error = m; return -1; };
    if (const char* why = verify_refuses(batch, n_drafts, vocab)) return fail(why);
    if (dtype > GEHTP_DT_F16) return fail("verify drafts: element type is GEHTP_DT_F32, GEHTP_DT_BF16 or GEHTP_DT_F16");
    if (!(temperature >= 0.0) || !std::isfinite(temperature) || (temperature > 0.0 && (temperature < 1e-4 || temperature > 1e4)))
        return fail("verify drafts: temperature is 0 or between 1e-4 and 1e4");
    const bool greedy = temperature == 0.0;
    if (!target_dev || !accepted_dev || !out_dev || !workspace_dev || (n_drafts && !tokens_dev) || (!greedy && !uniforms_dev)) return fail("verify drafts: null pointer");
    const void* draft = greedy || !n_drafts ? nullptr : draft_dev;
    if (target_stride < vocab || (draft && draft_stride < vocab)) return fail("verify drafts: rows are as long as the vocabulary at least");
    const uintptr_t el = dtype == GEHTP_DT_F32 ? 3u : 1u;
    if ((((uintptr_t)target_dev) | ((uintptr_t)draft)) & el) return fail("verify drafts: logits lie on boundaries of their type");
    if ((((uintptr_t)tokens_dev) | ((uintptr_t)n_drafts_dev) | ((uintptr_t)uniforms_dev) | ((uintptr_t)accepted_dev) | ((uintptr_t)out_dev)) & 3u)
        return fail("verify drafts: tokens, counts, uniforms and outputs lie on 4-byte boundaries");
    if ((uintptr_t)workspace_dev & 255u) return fail("verify drafts: the workspace lies on a 256-byte boundary");
    const size_t need = gehtp_verify_drafts_workspace(batch, n_drafts, vocab);
    if (workspace_bytes < need) {
        char m[128];
        std::snprintf(m, sizeof m, "verify drafts: needs %zu bytes of workspace, got %zu", need, workspace_bytes);
        return fail(m);
    }
    if (!on_this_device(target_dev, "verify drafts: target") || (draft && !on_this_device(draft, "verify drafts: draft")) ||
        (n_drafts && !on_this_device(tokens_dev, "verify drafts: tokens")) || (n_drafts_dev && !on_this_device(n_drafts_dev, "verify drafts: n_drafts")) ||
        (!greedy && !on_this_device(uniforms_dev, "verify drafts: uniforms")) || !on_this_device(accepted_dev, "verify drafts: accepted") ||
        !on_this_device(out_dev, "verify drafts: out") || !on_this_device(workspace_dev, "verify drafts: workspace"))
        return -1;
    VerifyArgs a{};
    a.target = target_dev; a.draft = draft; a.tokens = tokens_dev; a.n_drafts = n_drafts_dev; a.uniforms = uniforms_dev;
    a.accepted = accepted_dev; a.out = out_dev; a.batch = batch; a.n = n_drafts; a.vocab = vocab;
    cut_rows(batch, n_drafts, vocab, &a.piece, &a.pieces);
    a.t_stride = target_stride; a.d_stride = draft_stride;
    a.inv = greedy ? 0.0 : 1.0 / temperature;
    a.part = (float2*)workspace_dev;
    if (!k_verify_drafts((cudaStream_t)stream, a, dtype, greedy)) {
        const cudaError_t e = cudaGetLastError();
        return fail(e == cudaSuccess ? "verify drafts: launch refused" : cudaGetErrorString(e));
    }
    return 0;
}
