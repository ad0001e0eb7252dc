// Drafted tokens held against the target's probabilities, from given random numbers.
//
//   p_i = softmax(target_i / T), q_i = softmax(draft_i / T); without draft logits q_i is 1 at the drafted token
//   draft i is accepted while u_i q_i(x_i) < p_i(x_i)
//   the token behind the accepted ones: the first v whose sum of r over 0 .. v is above u_n times the sum of all r, where
//   r = max(p_i - q_i, 0) at the first place i that was not accepted (p_i where the rows are alike: a sum below 1e-12), r = p_n when all were
//   T = 0: x_i is accepted while it is the lowest place of the largest logit, and the token behind is that place
//
// verify_rows_kernel: maximum and sum of 2^((x - maximum) k), k = log2(e) / T, of pieces of the rows, a warp to a piece, in fp32: within some
// 2^-20, which is what the tests of acceptance go by. Rows that are there are counted first, and cut so that every warp has a like share.
// verify_choose_kernel: several CTAs per sequence decide, each for itself, how many are accepted, and draw the token behind them. A draw
// that ends next to the border of two tokens has to go to the right one, and there are as many borders as tokens: this one row
// is taken in 64 bits. Every warp has a stretch of the vocabulary; the CTA that comes last sees from the stretches' sums in which
// one the draw ends, and walks it.
// r needs the sums of p and q, which are not known in 64 bits before the row has been read: with c0 = sum q / sum p in fp32 in the place of the
// true c, one pass gives sum(e_p - c0 e_q) and sum(e_q) over the tokens where e_p > c0 e_q, and so sum(e_p - c e_q) = the first -
// (c - c0) times the second; tokens whose e_p / e_q lies between c0 and c (some 2^-22 wide) are off by no more than that width
// squared. Where p and q are so alike that this could show (a sum below 2^-10) the row is read once more with the true c.
#include <cooperative_groups.h>
#include <climits>
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

constexpr uint32_t MAX_DRAFTS = 64, MAX_SPLITS = 64;
constexpr int RT = 256, CT = 256, WARPS = CT / 32;
constexpr int CL = 8, GT = 512;             // T = 0 in one launch: CTAs of a cluster, their threads
constexpr uint32_t MAX_ROWS = 16;           // and the rows that it takes

struct VerifyArgs {
    const void *target, *draft;             // draft NULL: drafts without probabilities (and always with T = 0)
    const int32_t *tokens, *n_drafts;
    const float* uniforms;
    int32_t *accepted, *out;
    uint32_t batch, n, vocab;
    size_t t_stride, d_stride;
    double inv;                             // 1 / T
    uint32_t splits;                        // CTAs that share a sequence's draw
    uint32_t* done;                         // [batch] of them that are through; zeros when the second kernel starts
    double4* sums;                          // [batch][splits * WARPS] of the stretches
    uint32_t* base;                         // where n_drafts is given: [batch] first row of every sequence, behind them the pieces of a row
    uint32_t pieces;                        // where it is not
    float2* part;                           // [rows that are there][pieces] {maximum, sum}; T = 0: {maximum, its place}
};

struct El32 { typedef float T; static constexpr int V = 4; static __device__ float f(float x) { return x; } };
struct ElBf { typedef uint16_t T; static constexpr int V = 8; static __device__ float f(uint16_t x) { return bf2f(x); } };
struct ElHf { typedef uint16_t T; static constexpr int V = 8; static __device__ float f(uint16_t x) { return h2f(x); } };

// V logits from a 16-byte boundary on
template <class E>
__device__ __forceinline__ void unpack_logits(const uint4& v, float (&x)[E::V]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (E::V == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = E::f((typename E::T)(w[i] & 0xffffu)); x[2 * i + 1] = E::f((typename E::T)(w[i] >> 16)); }
    }
}
// (ordinary loads: a read-only one could be moved ahead of the wait for the kernel that writes the logits)
// V logits from place e on: in one load where they lie in the row and on a boundary; places outside the row are -inf
template <class E>
__device__ __forceinline__ void load_logits(const typename E::T* row, int64_t e, int64_t end, float (&x)[E::V]) {
    const typename E::T* p = row + e;
    if (e >= 0 && e + E::V <= end && ((uintptr_t)p & 15u) == 0) {
        unpack_logits<E>(__ldcg((const uint4*)p), x);
    } else {
#pragma unroll
        for (int i = 0; i < E::V; i++) x[i] = e + i >= 0 && e + i < end ? E::f(p[i]) : -INFINITY;
    }
}
// logits between the row's start and the last 16-byte boundary at or in front of it
template <class E>
__device__ __forceinline__ int lead(const typename E::T* row) { return (int)(((uintptr_t)row & 15u) / sizeof(typename E::T)); }

// 2^((x - m) k) in 64 bits: (x - m) k split into 32nds and at most half a 32nd; 2^that by a table of the 32 and the interpolation of degree 4 at
// the Chebyshev points of [-1/64, 1/64] (within 2^-43): nine 64-bit operations, of which 64 a cycle and SM run, where degree 9 over
// [-1/2, 1/2] takes thirteen. The difference comes first: products of numbers far from 0, as masks leave them, are rounded by more than it is. 0
// below 2^-1000 (its border rounded up: a number just below that is further down where neighbouring logits are) and for -inf.
struct Power64 {
    const double* table;                                      // 2^(j / 32)
    double k, m;
    float floor;
    __device__ __forceinline__ Power64(const double* table_, double k_, float m_) : table(table_), k(k_), m(m_) { floor = __double2float_ru(m - 1000.0 / k); }
    __device__ __forceinline__ double operator()(float x) const {
        const double d = (double)fmaxf(x, floor) - m, magic = 211106232532992.0 /* 1.5 * 2^47 */, n = fma(d, k, magic), f = fma(d, k, magic - n);
        const int i = __double2loint(n);                      // d k in 32nds
        double v = 0.009618176115571158;
        v = fma(v, f, 0.055504515573860415);
        v = fma(v, f, 0.24022650695623157);
        v = fma(v, f, 0.6931471805351095);
        v = fma(v, f, 1.0) * table[i & 31];
        const double e = __hiloint2double(__double2hiint(v) + ((i >> 5) << 20), __double2loint(v));
        return x >= floor ? e : 0.0;
    }
};

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

template <bool GREEDY>
__device__ __forceinline__ float2 together(float2 a, float2 b, float k) {
    if (GREEDY) return ahead(b.x, __float_as_int(b.y), a.x, __float_as_int(a.y)) ? b : a;
    return join(a, b, k);
}
// Parts of a row in N neighbouring lanes together (N a power of two); every one of them has the result.
template <bool GREEDY, int N>
__device__ __forceinline__ float2 join_lanes(float2 x, float k) {
#pragma unroll
    for (int o = N / 2; o; o >>= 1) x = together<GREEDY>(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)), k);
    return x;
}

constexpr int AHEAD = 4;                    // loads of a thread in flight

// {maximum, sum of 2^((x - maximum) k)} - GREEDY: {maximum, its place} - of the logits first .. end, by one warp; every lane has it.
// first is on a 16-byte boundary, or in front of the row by less than a vector.
template <class E, bool GREEDY>
__device__ __forceinline__ float2 part_of_row(const typename E::T* p, int64_t first, int64_t end, float k) {
    const uint32_t lane = threadIdx.x & 31;
    float2 best = make_float2(-INFINITY, 0.0f);
    int place = INT_MAX;
    bool odd = false;                                                // GREEDY: some logit is no number
    constexpr int64_t STEP = 32 * E::V;
    // N vectors of places e, e + STEP, ... together: one look at the maximum
    auto take = [&](const auto& x, int64_t e) {
        constexpr int N = sizeof(x) / sizeof(float);
        if (GREEDY) {
#pragma unroll
            for (int j = 0; j < N; j++) {                            // a lane's places ascend: the first of equal ones stays
                odd |= x[j] != x[j];
                if (x[j] > best.x) { best.x = x[j]; place = (int)(e + (j / E::V) * STEP + j % E::V); }
            }
        } else {
            float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int j = 4; j < N; j++) m[j & 3] = fmaxf(m[j & 3], x[j]);
            m[0] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            if (m[0] > best.x) {
                best.y = best.x == -INFINITY ? best.y : best.y * sm100::ex2((best.x - m[0]) * k);
                best.x = m[0];
            }
            const float off = best.x == -INFINITY ? 0.0f : best.x;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < N; j++) sum[j & 3] += sm100::ex2((x[j] - off) * k);
            best.y += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
    };
    int64_t e = first + lane * E::V;
    auto edge = [&] {                                                // what may have ends of the row among it
        uint4 w[AHEAD];
        float x[AHEAD * E::V];
#pragma unroll
        for (int u2 = 0; u2 < AHEAD; u2++) {                         // whole vectors first, all of them under way together
            const int64_t at = e + u2 * STEP;
            w[u2] = make_uint4(0u, 0u, 0u, 0u);
            if (at >= 0 && at + E::V <= end) w[u2] = __ldcg((const uint4*)(p + at));
        }
#pragma unroll
        for (int u2 = 0; u2 < AHEAD; u2++) {
            const int64_t at = e + u2 * STEP;
            float y[E::V];
            unpack_logits<E>(w[u2], y);
            if (at < 0 || at + E::V > end) {
#pragma unroll
                for (int i = 0; i < E::V; i++) y[i] = at + i >= 0 && at + i < end ? E::f(p[at + i]) : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < E::V; j++) x[u2 * E::V + j] = y[j];
        }
        take(x, e);
        e += AHEAD * STEP;
    };
    if (first < 0 && end > 0) edge();
    for (; e + (AHEAD - 1) * STEP + E::V <= end; e += AHEAD * STEP) {
        uint4 w[AHEAD];
        float x[AHEAD * E::V];
#pragma unroll
        for (int u2 = 0; u2 < AHEAD; u2++) w[u2] = __ldcg((const uint4*)(p + e + u2 * STEP));
#pragma unroll
        for (int u2 = 0; u2 < AHEAD; u2++) {
            float y[E::V];
            unpack_logits<E>(w[u2], y);
#pragma unroll
            for (int j = 0; j < E::V; j++) x[u2 * E::V + j] = y[j];
        }
        take(x, e);
    }
    while (e < end) edge();
    __syncwarp();
    if (GREEDY) {
        if (odd) { best.x = NAN; place = 0; }
        best.y = __int_as_float(place);
    }
    return join_lanes<GREEDY, 32>(best, k);
}

// Rows that are there, sequence by sequence: its target rows, then its draft rows.
__device__ __forceinline__ uint32_t rows_of(const VerifyArgs& A, uint32_t drafts) { return drafts * (A.draft ? 2 : 1) + 1; }

// Pieces of a row, `length` logits each but for what lies between a boundary and the row's start: 1024 at least; one to a warp of four
// CTAs an SM where that makes eight pieces or more, else 16 to 24, so that the last turn of the warps is a small part of all. (64 sequences
// with up to 7 drafts, 151936 tokens: 35 us; pieces of 8192 for whatever rows there are 42.5.)
struct Cut { uint32_t pieces, length; };
constexpr uint32_t ROW_WARPS = 148 * 4 * (RT / 32), MIN_PIECE = 1024, MOST_PIECES = 24;
__host__ __device__ inline Cut cut_rows(uint32_t vocab, uint32_t rows) {
    const uint32_t places = vocab + 7;                             // up to seven in front of the first boundary
    uint32_t pieces = ROW_WARPS / rows;
    if (pieces < 8) {
        pieces = (16 * rows + ROW_WARPS - 1) / ROW_WARPS * ROW_WARPS / rows;
        pieces = pieces < MOST_PIECES ? pieces : MOST_PIECES;
    }
    Cut c;
    c.length = ((places + pieces - 1) / pieces + 255) & ~255u;
    c.length = c.length > MIN_PIECE ? c.length : MIN_PIECE;
    c.pieces = (places + c.length - 1) / c.length;
    return c;
}

// A warp to a piece, in turns where there are more.
template <class E, bool GREEDY>
__global__ void __launch_bounds__(RT, 4) verify_rows_kernel(const VerifyArgs A) {
    extern __shared__ uint32_t base[];                               // [batch + 1] where n_drafts is given
    __shared__ uint32_t ends[RT / 32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, every = rows_of(A, A.n);
    pdl_wait();
    pdl_release();
    if (A.n_drafts) {
        const uint32_t per = (A.batch + RT - 1) / RT, from = min(A.batch, threadIdx.x * per), to = min(A.batch, from + per);
        uint32_t mine = 0, x;
        for (uint32_t b = from; b < to; b++) mine += rows_of(A, drafts_of(A, b));
        x = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        if (lane == 31) ends[warp] = x;
        __syncthreads();
        for (uint32_t w = 0; w < warp; w++) x += ends[w];
        if (threadIdx.x == RT - 1) base[A.batch] = x;
        x -= mine;
        for (uint32_t b = from; b < to; b++) { base[b] = x; x += rows_of(A, drafts_of(A, b)); }
        __syncthreads();
        if (blockIdx.x == 0)
            for (uint32_t b = threadIdx.x; b <= A.batch; b += RT) A.base[b] = b < A.batch ? base[b] : cut_rows(A.vocab, base[b]).pieces;
    }
    if (!GREEDY && blockIdx.x == 0)
        for (uint32_t b = threadIdx.x; b < A.batch; b += RT) A.done[b] = 0;
    const uint32_t rows = A.n_drafts ? base[A.batch] : A.batch * every;
    const Cut cut = cut_rows(A.vocab, rows);
    const float k = (float)(A.inv * 1.4426950408889634);
    for (uint32_t it = blockIdx.x * (RT / 32) + warp; it < rows * cut.pieces; it += gridDim.x * (RT / 32)) {
        const uint32_t r = it / cut.pieces, piece = it % cut.pieces;
        uint32_t b = 0, first_row, next;
        if (A.n_drafts) {
            for (uint32_t n = A.batch; n > 1;) {                     // the last sequence that begins at r or in front of it
                const uint32_t half = n / 2;
                if (base[b + half] <= r) b += half;
                n -= half;
            }
            first_row = base[b];
            next = base[b + 1];
        } else {
            b = r / every;
            first_row = b * every;
            next = first_row + every;
        }
        const uint32_t targets = A.draft ? (next - first_row + 1) / 2 : next - first_row, i = r - first_row;
        const typename E::T* p = i < targets ? (const typename E::T*)A.target + ((size_t)b * (A.n + 1) + i) * A.t_stride
                                             : (const typename E::T*)A.draft + ((size_t)b * A.n + i - targets) * A.d_stride;
        const int64_t from = (int64_t)piece * cut.length - lead<E>(p);
        const float2 best = part_of_row<E, GREEDY>(p, from, min((int64_t)A.vocab, from + cut.length), k);
        if (lane == 0) A.part[it] = best;
    }
}

// A row's parts together, by one warp.
template <bool GREEDY>
__device__ __forceinline__ float2 whole_row(const float2* part, uint32_t pieces, float k) {
    float2 x = make_float2(-INFINITY, GREEDY ? __int_as_float(INT_MAX) : 0.0f);
    for (uint32_t i = threadIdx.x & 31; i < pieces; i += 32) x = together<GREEDY>(x, part[i], k);
    return join_lanes<GREEDY, 32>(x, k);
}
__device__ __forceinline__ bool sound(float2 x) { return x.y > 0.0f && isfinite(x.y) && isfinite(x.x); }

// Sums over the CTA: of all threads, and of those in front of each.
struct BlockScan {
    double warp[WARPS];
    double2 pair[WARPS];
    __device__ __forceinline__ double2 sums(double2 v) {
        v.x = warp_sum_d(v.x);
        v.y = warp_sum_d(v.y);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) pair[threadIdx.x >> 5] = v;
        __syncthreads();
        double2 t = make_double2(0.0, 0.0);
#pragma unroll
        for (int i = 0; i < WARPS; i++) { t.x += pair[i].x; t.y += pair[i].y; }
        return t;
    }
    __device__ __forceinline__ double before(double v, double* total) {
        double x = v;
        for (int o = 1; o < 32; o <<= 1) {
            const double z = __shfl_up_sync(0xffffffffu, x, o);
            if ((threadIdx.x & 31) >= (uint32_t)o) x += z;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 31) warp[threadIdx.x >> 5] = x;
        __syncthreads();
        double t = 0.0, front = 0.0;
#pragma unroll
        for (int i = 0; i < WARPS; i++) { if (i == (int)(threadIdx.x >> 5)) front = t; t += warp[i]; }
        *total = t;
        return front + (x - v);
    }
};

struct DrawShared {
    BlockScan scan;
    int first, last, is_last;
    double front;
    double table[32];                                         // of Power64
};

// The lowest place of `hit` (a place or INT_MAX) over the CTA, and the sum in front of it.
__device__ __forceinline__ void lowest(DrawShared& S, int hit, double front) {
    if (threadIdx.x == 0) S.first = INT_MAX;
    __syncthreads();
    if (hit != INT_MAX) atomicMin(&S.first, hit);
    __syncthreads();
    if (hit != INT_MAX && S.first == hit) S.front = front;
    __syncthreads();
}

// The token that a draw from r = max(p - q, 0) (from p without q, or where they are alike) ends in; `away` is never drawn, and comes back
// where nothing else has a weight. The last CTA of a sequence writes it.
template <class E>
__device__ __forceinline__ void draw(const VerifyArgs& A, uint32_t b, const typename E::T* p, const typename E::T* q, float2 rp, float2 rq, double k, double u, int away,
                                     DrawShared& S, int32_t* to_) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stretches = A.splits * WARPS;
    const int64_t vocab = A.vocab, p_lead = lead<E>(p), vecs = (vocab + p_lead + E::V - 1) / E::V;
    const Power64 ep(S.table, k, rp.x), eq(S.table, k, rq.x);
    const double c0 = q ? (double)(rp.y / rq.y) : 0.0;
    {
        const int64_t mine = blockIdx.x * WARPS + warp, from = vecs * mine / stretches, to = vecs * (mine + 1) / stretches;
        double4 v = make_double4(0.0, 0.0, 0.0, 0.0);         // sums of e_p, e_q; e_p - c0 e_q and e_q where the former is positive
        for (int64_t j = from + lane; j < to; j += 32) {
            const int64_t e = j * E::V - p_lead;
            float x[E::V], y[E::V];
            load_logits<E>(p, e, vocab, x);
            if (q) {
                load_logits<E>(q, e, vocab, y);
#pragma unroll
                for (int i = 0; i < E::V; i++) {
                    const double a = ep(x[i]), d = eq(y[i]), r = fma(-c0, d, a);
                    const bool more = __double2hiint(r) > 0;
                    v.x += a;
                    v.y += d;
                    v.z += more ? r : 0.0;
                    v.w += more ? d : 0.0;
                }
            } else {
#pragma unroll
                for (int i = 0; i < E::V; i++) v.x += e + i == away ? 0.0 : ep(x[i]);
            }
        }
        v.x = warp_sum_d(v.x);
        if (q) { v.y = warp_sum_d(v.y); v.z = warp_sum_d(v.z); v.w = warp_sum_d(v.w); }
        if (lane == 0) {
            A.sums[(size_t)b * stretches + mine] = v;
            __threadfence();
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) S.is_last = atomicAdd(&A.done[b], 1u) + 1 == A.splits;
    __syncthreads();
    if (!S.is_last) return;
    __threadfence();
    // ---- the last: weights of the stretches, two to a thread
    static_assert(MAX_SPLITS * WARPS <= 2 * CT, "two stretches to a thread");
    const double4* sums = A.sums + (size_t)b * stretches;
    double4 v[2];
    double w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t at = threadIdx.x * 2 + i;
        v[i] = make_double4(0.0, 0.0, 0.0, 0.0);
        if (at < stretches) { const double2 *x = (const double2*)(sums + at), lo = __ldcg(x), hi = __ldcg(x + 1); v[i] = make_double4(lo.x, lo.y, hi.x, hi.y); }
        w[i] = v[i].x;
    }
    double c = 0.0;
    bool less = q != nullptr;                                 // the weights are p - q
    // e_p - c e_q with the product rounded on its own: equal rows leave 0
    auto rest = [&](float x, float y) { return fmax(ep(x) - __dmul_rn(c, eq(y)), 0.0); };
    double total, front, tp = 0.0;
    if (less) {
        const double2 t = S.scan.sums(make_double2(v[0].x + v[1].x, v[0].y + v[1].y));
        tp = t.x;
        c = t.x / t.y;
#pragma unroll
        for (int i = 0; i < 2; i++) w[i] = fmax(fma(c0 - c, v[i].w, v[i].z), 0.0);
    }
    front = S.scan.before(w[0] + w[1], &total);
    if (less && total < 0x1p-10 * tp) {                       // p and q nearly alike: once more with the true c
        __shared__ double again[MAX_SPLITS * WARPS];
        for (uint32_t at = warp; at < stretches; at += WARPS) {
            const int64_t from = vecs * at / stretches, to = vecs * (at + 1) / stretches;
            double r = 0.0;
            for (int64_t j = from + lane; j < to; j += 32) {
                const int64_t e = j * E::V - p_lead;
                float x[E::V], y[E::V];
                load_logits<E>(p, e, vocab, x);
                load_logits<E>(q, e, vocab, y);
#pragma unroll
                for (int i = 0; i < E::V; i++) r += rest(x[i], y[i]);
            }
            r = warp_sum_d(r);
            if (lane == 0) again[at] = r;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; i++) w[i] = threadIdx.x * 2 + i < stretches ? again[threadIdx.x * 2 + i] : 0.0;
        front = S.scan.before(w[0] + w[1], &total);
        if (total <= 1e-12 * tp) {                            // what the roundings of two sums leave of equal rows
            less = false;
            w[0] = v[0].x; w[1] = v[1].x;
            front = S.scan.before(w[0] + w[1], &total);
        }
    }
    const double goal = fmax(u * total, 0.0);
    // the first stretch whose end is above the goal; a draw of 1 and above ends in the last that has a weight
    if (threadIdx.x == 0) S.last = -1;
    __syncthreads();
    if (w[0] > 0.0 || w[1] > 0.0) atomicMax(&S.last, (int)threadIdx.x * 2 + (w[1] > 0.0 ? 1 : 0));
    int hit = INT_MAX;
    if (w[0] > 0.0 && front + w[0] > goal) hit = threadIdx.x * 2;
    else if (w[1] > 0.0 && front + w[0] + w[1] > goal) hit = threadIdx.x * 2 + 1;
    lowest(S, hit, hit & 1 ? front + w[0] : front);
    if (S.first == INT_MAX) {
        if (S.last < 0) {
            if (threadIdx.x == 0) *to_ = away;                // all of p lay on the rejected token
            return;
        }
        lowest(S, (int)threadIdx.x == S.last / 2 ? S.last : INT_MAX, S.last & 1 ? front + w[0] : front);
    }
    // The token in that stretch. What p - q leaves of like tokens is the rounding of two sums, so a stretch may have a weight and no token with
    // one (at the ends of the draw, where the goal is 0 or the whole sum): then the next stretch's first token, else one in front of it.
    const int begin = S.first;
    double upto = S.front;
    for (int at = begin, way = 1; ; at += way) {
        if (at == (int)stretches) { at = begin - 1; way = -1; }
        if (at < 0) break;                                    // not reached: some token has a weight
        const int64_t from = vecs * at / stretches, to = vecs * (at + 1) / stretches;
        const double end = at == begin ? goal : way > 0 ? -1.0 : INFINITY;
        __syncthreads();
        if (threadIdx.x == 0) { S.last = -1; S.first = INT_MAX; }
        for (int64_t j0 = from; j0 < to; j0 += CT) {
            const int64_t j = j0 + threadIdx.x, e = j * E::V - p_lead;
            float x[E::V], y[E::V];
            double r[E::V], sum = 0.0, all;
            if (j < to) {
                load_logits<E>(p, e, vocab, x);
                if (less) load_logits<E>(q, e, vocab, y);
            }
#pragma unroll
            for (int i = 0; i < E::V; i++) {
                r[i] = j >= to || e + i == away ? 0.0 : less ? rest(x[i], y[i]) : ep(x[i]);
                sum += r[i];
            }
            double s = upto + S.scan.before(sum, &all);
            int here = INT_MAX, some = -1;
#pragma unroll
            for (int i = 0; i < E::V; i++) {
                s += r[i];
                if (r[i] > 0.0) {
                    some = (int)(e + i);
                    if (here == INT_MAX && s > end) here = some;
                }
            }
            if (some >= 0) atomicMax(&S.last, some);
            lowest(S, here, 0.0);
            if (S.first != INT_MAX) break;
            upto += all;
        }
        __syncthreads();
        // the stretch's sum was above the goal: its last possible token at the latest
        const int token = S.first != INT_MAX ? S.first : S.last;
        if (token >= 0) {
            if (threadIdx.x == 0) *to_ = token;
            return;
        }
    }
    if (threadIdx.x == 0) *to_ = -1;
}

// What a sequence gets: `a` accepted drafts, -1 behind the token that follows them.
__device__ __forceinline__ void write_accepted(const VerifyArgs& A, uint32_t b, uint32_t a) {
    int32_t* out = A.out + (size_t)b * (A.n + 1);
    if (threadIdx.x == 0) A.accepted[b] = (int)a;
    for (uint32_t i = threadIdx.x; i <= A.n; i += blockDim.x)
        if (i != a) out[i] = i < a ? A.tokens[(size_t)b * A.n + i] : -1;
}

// grid: (CTAs of a sequence, sequences)
template <class E, bool GREEDY>
__global__ void __launch_bounds__(CT, 4) verify_choose_kernel(const VerifyArgs A) {
    __shared__ DrawShared shared;
    __shared__ uint8_t pass[MAX_DRAFTS];
    __shared__ float2 rows[MAX_DRAFTS + 1][2];                    // {maximum, sum} of target and draft rows
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.y;
    pdl_wait();
    pdl_release();
    const uint32_t nd = drafts_of(A, b);
    if (!GREEDY && threadIdx.x < 32) shared.table[threadIdx.x] = exp2(threadIdx.x / 32.0);
    const typename E::T *target = (const typename E::T*)A.target + (size_t)b * (A.n + 1) * A.t_stride, *draft = (const typename E::T*)A.draft + (size_t)b * A.n * A.d_stride;
    const double k = A.inv * 1.4426950408889634;
    const uint32_t base = A.n_drafts ? A.base[b] : b * rows_of(A, A.n);
    const uint32_t pieces = A.n_drafts ? A.base[A.batch] : A.pieces;
    const float2* part = A.part + (size_t)base * pieces;
    // ---- which drafts pass; the row behind the last one is looked at beside them
    for (uint32_t i = warp; i <= nd; i += WARPS) {
        const int x = i < nd ? A.tokens[(size_t)b * A.n + i] : -1;
        const bool in = x >= 0 && (uint32_t)x < A.vocab;
        const double lp = !GREEDY && in ? (double)E::f(target[i * A.t_stride + x]) : 0.0, lq = !GREEDY && in && A.draft ? (double)E::f(draft[i * A.d_stride + x]) : 0.0;
        const float2 p = whole_row<GREEDY>(part + (size_t)i * pieces, pieces, (float)k);
        float2 q = make_float2(NAN, NAN);
        bool ok = i < nd;
        if (GREEDY) {
            ok = ok && isfinite(p.x) && x == __float_as_int(p.y);
        } else if (ok) {
            double px = 0.0, qx = 1.0;
            ok = sound(p);
            if (ok && in) px = exp2((lp - p.x) * k) / p.y;
            if (A.draft) {
                q = whole_row<false>(part + (size_t)(nd + 1 + i) * pieces, pieces, (float)k);
                ok = ok && sound(q);
                qx = ok && in ? exp2((lq - q.x) * k) / q.y : 0.0;
            }
            ok = ok && (double)A.uniforms[(size_t)b * (A.n + 1) + i] * qx < px;
        }
        if (lane == 0) {
            if (i < nd) pass[i] = ok;
            rows[i][0] = p; rows[i][1] = q;
        }
    }
    __syncthreads();
    uint32_t a = 0;
    while (a < nd && pass[a]) a++;
    const bool rejected = a < nd;
    int32_t* token = A.out + (size_t)b * (A.n + 1) + a;
    if (blockIdx.x == 0) write_accepted(A, b, a);
    // ---- the row behind the accepted ones
    const float2 rp = rows[a][0], rq = rows[a][1];
    if constexpr (GREEDY) {
        if (threadIdx.x == 0) *token = isfinite(rp.x) ? __float_as_int(rp.y) : -1;
    } else {
        if (!sound(rp)) {                                   // a row without a distribution, for all CTAs of the sequence
            if (blockIdx.x == 0 && threadIdx.x == 0) *token = -1;
            return;
        }
        const int away = rejected && !A.draft ? A.tokens[(size_t)b * A.n + a] : -1;
        const typename E::T *p = target + a * A.t_stride, *q = sound(rq) ? draft + a * A.d_stride : nullptr;   // a draft row without one takes nothing away
        draw<E>(A, b, p, q, rp, rq, k, (double)A.uniforms[(size_t)b * (A.n + 1) + A.n], away, shared, token);
    }
}

// T = 0 and few logits, in one launch: a cluster of eight CTAs to a sequence, a warp to a piece of a row. The CTAs' warps tell one another what
// they found, and the first CTA decides. A launch less is some 2 us of the host's time, which is what a small call costs: one
// sequence, four drafts, 32768 tokens 10.8 us against 13.5 call by call.
template <class E>
__global__ void __launch_bounds__(GT) verify_greedy_kernel(const VerifyArgs A) {
    constexpr uint32_t GW = GT / 32, ALL = CL * GW;
    __shared__ float2 parts[ALL], whole[MAX_ROWS];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = blockIdx.x / CL, mine = cluster.block_rank() * GW + warp;
    cluster_arrive();                                             // with the wait below: nothing is written to a CTA before it runs
    pdl_wait();
    pdl_release();
    const uint32_t nd = drafts_of(A, b), per = ALL / (nd + 1), r = mine / per;
    float2 v = make_float2(-INFINITY, __int_as_float(INT_MAX));
    if (r <= nd) {
        const typename E::T* p = (const typename E::T*)A.target + ((size_t)b * (A.n + 1) + r) * A.t_stride;
        const int64_t p_lead = lead<E>(p), vecs = ((int64_t)A.vocab + p_lead + E::V - 1) / E::V, at = mine % per;
        v = part_of_row<E, true>(p, vecs * at / per * E::V - p_lead, min((int64_t)A.vocab, vecs * (at + 1) / per * E::V - p_lead), 0.0f);
    }
    cluster_wait();
    if (lane == 0) *cluster.map_shared_rank(&parts[mine], 0) = v;
    cluster.sync();
    if (cluster.block_rank() != 0) return;
    if (warp <= nd) {
        const float2 x = whole_row<true>(parts + warp * per, per, 0.0f);
        if (lane == 0) whole[warp] = x;
    }
    __syncthreads();
    uint32_t a = 0;
    while (a < nd && isfinite(whole[a].x) && A.tokens[(size_t)b * A.n + a] == __float_as_int(whole[a].y)) a++;
    write_accepted(A, b, a);
    if (threadIdx.x == 0) A.out[(size_t)b * (A.n + 1) + a] = isfinite(whole[a].x) ? __float_as_int(whole[a].y) : -1;
}

const char* verify_refuses(uint32_t batch, uint32_t n, uint32_t vocab) {
    if (!batch || batch > 4096) return "verify drafts: 1 to 4096 sequences";
    if (n > MAX_DRAFTS) return "verify drafts: up to 64 drafts";
    if (!vocab || vocab > (1u << 30)) return "verify drafts: a vocabulary of 1 to 2^30";
    return nullptr;
}

// CTAs to a sequence's draw: four an SM over all sequences, while every thread has a vector of logits
uint32_t cut_draw(uint32_t batch, uint32_t vocab) {
    return std::max(1u, std::min({MAX_SPLITS, 148 * 4 / batch, vocab / (CT * 8)}));
}

struct Layout { size_t sums, base, part, total; };
Layout lay_out(uint32_t batch, uint32_t n, uint32_t vocab) {
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    Layout l;
    l.sums = up((size_t)batch * 4);
    l.base = l.sums + up((size_t)batch * cut_draw(batch, vocab) * WARPS * sizeof(double4));
    l.part = l.base + up((size_t)(batch + 1) * 4);
    // at most: one piece to a warp, or few to a row
    l.total = l.part + up((ROW_WARPS + (size_t)batch * (2 * n + 1) * std::min(MOST_PIECES, vocab / MIN_PIECE + 2)) * 8);
    return l;
}

template <class E, bool GREEDY>
bool launch_verify(cudaStream_t st, const VerifyArgs& a) {
    // one launch while a cluster's share is a megabyte at most and the clusters find room at once
    if (GREEDY && a.n < MAX_ROWS && (size_t)(a.n + 1) * a.vocab * sizeof(typename E::T) <= (1u << 20) && a.batch <= 148 / CL) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a.batch * CL); cfg.blockDim = dim3(GT); cfg.stream = st;
        g_launches++;
        return launch_pdl_cluster(verify_greedy_kernel<E>, cfg, dim3(CL, 1, 1), a) == cudaSuccess;
    }
    const uint64_t most = (uint64_t)a.batch * (a.n * (a.draft ? 2 : 1) + 1) * (a.vocab / MIN_PIECE + 1), warps = std::min<uint64_t>(most, ROW_WARPS);
    g_launches += 2;
    if (launch_pdl(verify_rows_kernel<E, GREEDY>, dim3((uint32_t)((warps + RT / 32 - 1) / (RT / 32))), dim3(RT), a.n_drafts ? (a.batch + 1) * 4 : 0, st, a) != cudaSuccess) return false;
    return launch_pdl(verify_choose_kernel<E, GREEDY>, dim3(GREEDY ? 1 : a.splits, a.batch), dim3(CT), 0, st, a) == cudaSuccess;
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
    return lay_out(batch, n_drafts, vocab).total;
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
    // a sequence's outputs are written while other CTAs read its inputs
    const size_t each = (size_t)batch * 4, all = each * n_drafts;
    for (const void* in : {(const void*)tokens_dev, (const void*)n_drafts_dev, (const void*)uniforms_dev}) {
        const size_t bytes = in == n_drafts_dev ? each : in == tokens_dev ? all : all + each;
        if (!apart(in, bytes, accepted_dev, each) || !apart(in, bytes, out_dev, all + each)) return fail("verify drafts: an output overlaps an input");
    }
    if ((uintptr_t)workspace_dev & 255u) return fail("verify drafts: the workspace lies on a 256-byte boundary");
    const Layout l = lay_out(batch, n_drafts, vocab);
    if (workspace_bytes < l.total) {
        char m[128];
        std::snprintf(m, sizeof m, "verify drafts: needs %zu bytes of workspace, got %zu", l.total, workspace_bytes);
        return fail(m);
    }
    if (!on_this_device(target_dev, "verify drafts: target") || (draft && !on_this_device(draft, "verify drafts: draft")) ||
        (n_drafts && !on_this_device(tokens_dev, "verify drafts: tokens")) || (n_drafts_dev && !on_this_device(n_drafts_dev, "verify drafts: n_drafts")) ||
        (!greedy && !on_this_device(uniforms_dev, "verify drafts: uniforms")) || !on_this_device(accepted_dev, "verify drafts: accepted") ||
        !on_this_device(out_dev, "verify drafts: out") || !on_this_device(workspace_dev, "verify drafts: workspace"))
        return -1;
    const size_t rows = (size_t)batch * (n_drafts + 1), size = dtype == GEHTP_DT_F32 ? 4 : 2;
    if (!all_apart({{accepted_dev, each}, {out_dev, rows * 4}, {workspace_dev, l.total}},
                   {{target_dev, ((rows - 1) * target_stride + vocab) * size}, {draft, draft ? (((size_t)batch * n_drafts - 1) * draft_stride + vocab) * size : 0},
                    {tokens_dev, all}, {n_drafts_dev, n_drafts_dev ? each : 0}, {uniforms_dev, greedy ? 0 : rows * 4}}))
        return fail("verify drafts: an output or the workspace overlaps another operand");
    VerifyArgs a{};
    a.target = target_dev; a.draft = draft; a.tokens = tokens_dev; a.n_drafts = n_drafts_dev; a.uniforms = uniforms_dev;
    a.accepted = accepted_dev; a.out = out_dev; a.batch = batch; a.n = n_drafts; a.vocab = vocab;
    a.pieces = cut_rows(vocab, batch * (n_drafts * (draft ? 2 : 1) + 1)).pieces;
    a.t_stride = target_stride; a.d_stride = draft_stride;
    a.inv = greedy ? 0.0 : 1.0 / temperature;
    unsigned char* ws = (unsigned char*)workspace_dev;
    a.splits = cut_draw(batch, vocab);
    a.done = (uint32_t*)ws; a.sums = (double4*)(ws + l.sums); a.base = (uint32_t*)(ws + l.base); a.part = (float2*)(ws + l.part);
    if (!k_verify_drafts((cudaStream_t)stream, a, dtype, greedy)) {
        const cudaError_t e = cudaGetLastError();
        return fail(e == cudaSuccess ? "verify drafts: launch refused" : cudaGetErrorString(e));
    }
    return 0;
}
