// Attention of a batch over a prefix that all its sequences share and a tail of each one's own:
//
//   out = sum_j p_j v_j,  p = softmax(scale q.k_j),  j over the prefix and over the tail positions the row sees
//
// Query t of a sequence (of q_len new tokens, the last positions of its tail) sees the tail up to its own position. The prefix is
// read once for all sequences: its keys meet the rows of all of them, rep query heads to a key head. Rows of one tail are few
// (q_len * rep). No row's result depends on a position that it does not see, whatever is cached there.
//
// Items of work: (row tile, key head, slice of the prefix) and (sequence, key head, slice of its tail). How a batch's tails are cut follows
// from their lengths, which lie on the device: every CTA works that out for itself. S and P stay in registers (mma.sync m16n8k16).
// shared_parts_kernel: an item to as many warps as it has 16 rows.
// shared_merge_kernel: partial results of a row together; where asked for, the weights of the tail positions.
#include <atomic>
#include <chrono>
#include <climits>
#include <cmath>
#include <cstdio>
#include "engine.h"
#include "launchers_batch.h"
#include "mma_bf16.cuh"
#include "sm100_attn.cuh"

namespace gehtp {

namespace {

constexpr uint32_t TILE = 64, MAX_BATCH = 1024, MAX_Q = 16, MAX_ROWS = 128;
constexpr uint32_t SMS = 148;

template <bool BF>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF) {
        mma_bf16(c, a, b0, b1);
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
template <bool BF>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if (BF) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*(const __half2*)&w);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF) return pack_bf2(a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}

// A score's weight beside a maximum. It meets the values as a word of 16 bits. Where that is fp16 it is made 2^LIFT times as large, which is still below 2^16, so
// that its 11 bits last down to 2^-29 of the row's largest, and a part of it to 2^-40; without, weights below 2^-25 were gone from the result
// though their sum was not. Sums and outputs give the factor back when they are written.
template <bool BF>
constexpr float LIFT = BF ? 0.0f : 15.0f;
template <bool BF>
__device__ __forceinline__ float weight(float s, float m) { return sm100::ex2(BF ? s - m : (s - m) + LIFT<BF>); }
template <bool BF>
constexpr float UNLIFT = BF ? 1.0f : 0x1p-15f;

__device__ __forceinline__ uint32_t tail_length(const SharedArgs& A, uint32_t b) { return (uint32_t)min(max(A.n_tail[b], 0), (int)A.nslots); }
// tail positions that all rows of a sequence see
__device__ __forceinline__ uint32_t common_length(const SharedArgs& A, uint32_t n) { return n + 1 > A.q_len ? n + 1 - A.q_len : 0; }

// Slices in front of each sequence's (cum[batch]: all of them) and positions to a slice, by one warp. Slices are as long as cuts
// the tails together into about t_slices, 64 positions at least and then in steps of 16 where one warp has an item; a sequence with any
// position has one at least.
__device__ uint32_t cut_tails(const SharedArgs& A, uint32_t* cum) {
    const uint32_t lane = threadIdx.x & 31, cut = A.q_len * A.rep <= 16 ? 16 : TILE;
    uint32_t tiles = 0;
    for (uint32_t b = lane; b < A.batch; b += 32) tiles += (common_length(A, tail_length(A, b)) + cut - 1) / cut;
    for (int o = 16; o; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    const uint32_t k = max(TILE / cut, (tiles + A.t_slices - 1) / A.t_slices);
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < A.batch; b0 += 32) {
        const uint32_t b = b0 + lane;
        uint32_t s = 0;
        if (b < A.batch) {
            const uint32_t n = tail_length(A, b), t = (common_length(A, n) + cut - 1) / cut;
            s = n ? max(1u, (t + k - 1) / k) : 0;
        }
        uint32_t x = s;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        if (b < A.batch) cum[b] = before + x - s;
        before += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) cum[A.batch] = before;
    return k * cut;
}

// What an item has to do: rows against keys, and the place of its partial results.
struct Item {
    bool tail, last;                       // last: it holds the end of a tail
    uint32_t h, rows, token0, from, to;    // key head; rows, their first token; positions
    uint32_t b, n, c;                      // of a tail: its sequence, its length, positions that all rows see
    size_t v_off, out;                     // from a key to its value, half of what lies between two keys; first partial row
    const uint16_t* kbase;
};

template <int HD>
__device__ __forceinline__ Item item_of(const SharedArgs& A, const uint32_t* cum, uint32_t k, uint32_t w, uint32_t prefix_items) {
    Item I;
    I.tail = w >= prefix_items;
    I.last = false;
    I.b = I.n = I.c = 0;
    if (!I.tail) {
        const uint32_t tile = w % A.p_tiles, u = w / A.p_tiles, s = u / A.kv_heads;
        I.h = u % A.kv_heads;
        I.token0 = tile * A.p_tokens;
        I.rows = min(A.p_tokens, A.batch * A.q_len - I.token0) * A.rep;
        I.from = s * A.p_len;
        I.to = min(A.n_prefix, I.from + A.p_len);
        I.v_off = (size_t)A.kv_heads * HD;
        I.kbase = A.prefix + (size_t)I.h * HD;
        I.out = (((size_t)tile * A.kv_heads + I.h) * A.p_slices + s) * (A.p_tokens * A.rep);
    } else {
        const uint32_t u = (w - prefix_items) / A.kv_heads;
        I.h = (w - prefix_items) % A.kv_heads;
        uint32_t b = 0, hi = A.batch;                              // cum[b] <= u < cum[b + 1]
        while (hi - b > 1) {
            const uint32_t mid = (b + hi) / 2;
            if (cum[mid] <= u) b = mid; else hi = mid;
        }
        I.b = b;
        I.n = tail_length(A, b);
        I.c = common_length(A, I.n);
        I.token0 = b * A.q_len;
        I.rows = A.q_len * A.rep;
        I.from = (u - cum[b]) * k;
        I.last = u + 1 == cum[b + 1];
        I.to = I.last ? I.n : I.from + k;
        I.v_off = (size_t)A.batch * A.kv_heads * HD;
        I.kbase = A.tail + ((size_t)b * A.kv_heads + I.h) * HD;
        I.out = A.p_rows() + ((size_t)u * A.kv_heads + I.h) * I.rows;
    }
    return I;
}

// 8x8 words of 16 bits, a row's pairs over four lanes, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// At most 8 rows against 16 positions at a time: the positions are the products' 16 rows and the item's rows their 8 columns, where rows as
// rows would leave half of every product, exponential and register to nobody. A lane has the rows 2 (lane % 4) and 1 more, at
// positions lane / 4 and 8 further. 32 sequences of 32 heads, tails of up to 2048 alone: 42.5 us, rows as rows 47.7; 16 of up to 1024 16.2 and 20.0.
template <bool BF, int HD>
struct Few {
    uint32_t q[HD / 16][2];
    float o[HD / 16][4], m[2], l[2];
    int lim[2];                                                       // the first position that a row does not see

    __device__ __forceinline__ void begin(const SharedArgs& A, const Item& I, uint32_t lane) {
        const uint32_t r = lane >> 2, q4 = lane & 3;
        const bool in = r < I.rows;
        const uint16_t* qp = A.q + (in ? (size_t)(I.token0 + r / A.rep) * A.q_stride + (size_t)(I.h * A.rep + r % A.rep) * HD : 0) + q4 * 2;
#pragma unroll
        for (int x = 0; x < HD / 16; x++) {
            q[x][0] = in ? *(const uint32_t*)(qp + x * 16) : 0u;
            q[x][1] = in ? *(const uint32_t*)(qp + x * 16 + 8) : 0u;
            o[x][0] = o[x][1] = o[x][2] = o[x][3] = 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            lim[e] = I.last ? min((int)I.to, (int)(I.n + (q4 * 2 + e) / A.rep + 1) - (int)A.q_len) : (int)I.to;
            m[e] = -INFINITY;
            l[e] = 0.0f;
        }
    }

    // kt, vt: shared addresses of 16 keys and their values; v: the values once more
    __device__ __forceinline__ void step(const SharedArgs& A, const Item& I, uint32_t p0, uint32_t kt, uint32_t vt, const unsigned char* v, uint32_t lane) {
        constexpr uint32_t ROW = HD * 2;
        const uint32_t g8 = lane >> 2, q4 = lane & 3;
        float s[4] = {};                                              // position g8 + 8 (e / 2), row 2 q4 + e % 2
        {
            const uint32_t r = (lane & 7) + ((lane >> 3) & 1) * 8;
            float s2[4] = {};
#pragma unroll
            for (int x = 0; x < HD / 16; x++) {
                uint32_t f[4];
                ldsm4(f, kt + r * ROW + (((2 * x + ((lane >> 4) & 1)) ^ (r & 7)) * 16));
                mma16<BF>(x & 1 ? s2 : s, f, q[x][0], q[x][1]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) s[e] += s2[e];
        }
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            s[e] = (int)(p0 + g8 + (e >> 1) * 8) < lim[e & 1] ? s[e] * A.sc : -INFINITY;
            mx[e & 1] = fmaxf(mx[e & 1], s[e]);
        }
        if (I.tail && A.scores) {
            float* sp = A.scores + (((size_t)I.b * A.kv_heads + I.h) * I.rows + q4 * 2) * A.nslots + p0 + g8;
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (q4 * 2 + (e & 1) < I.rows && p0 + g8 + (e >> 1) * 8 < I.to) sp[(size_t)(e & 1) * A.nslots + (e >> 1) * 8] = s[e];
        }
        if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int d = 4; d < 32; d *= 2) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], d));
                const float mn = fmaxf(m[e], mx[e]), f = mn > m[e] ? (m[e] == -INFINITY ? 0.0f : sm100::ex2(m[e] - mn)) : 1.0f;
                m[e] = mn;
                l[e] *= f;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) { o[j][e] *= f; o[j][2 + e] *= f; }
            }
        }
        const float off[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            s[e] = weight<BF>(s[e], off[e & 1]);
            l[e & 1] += s[e];
        }
        // as below: values that are no numbers, at positions that only some rows see
        bool odd = false;
        if (I.last && p0 + 16 > I.c && I.n > I.c) {
            constexpr uint32_t EXP = BF ? 0x7f807f80u : 0x7c007c00u;
#pragma unroll 1
            for (uint32_t e = lane; e < 2 * HD; e += 32)
                for (uint32_t u = 0; u < 4; u++) {
                    const uint32_t x = ((const uint32_t*)v)[e * 4 + u];
                    odd |= (x & EXP & 0xffffu) == (EXP & 0xffffu) || (x & EXP & 0xffff0000u) == (EXP & 0xffff0000u);
                }
            odd = __any_sync(0xffffffffu, odd);
        }
        if (odd) {
#pragma unroll 1
            for (uint32_t col = 0; col < 16; col++) {
                float p[2];
#pragma unroll
                for (int e = 0; e < 2; e++) p[e] = __shfl_sync(0xffffffffu, col < 8 ? s[e] : s[2 + e], (int)((col % 8) * 4 + q4));
#pragma unroll
                for (int j = 0; j < HD / 8; j++) {
                    const float x = unpack2<BF>(*(const uint16_t*)(v + col * ROW + ((j ^ (col & 7)) * 16) + g8 * 2)).x;
#pragma unroll
                    for (int e = 0; e < 2; e++)
                        if ((int)(p0 + col) < lim[e]) o[j / 2][j % 2 * 2 + e] = fmaf(p[e], x, o[j / 2][j % 2 * 2 + e]);
                }
            }
            return;
        }
        uint32_t hi[2], lo[2];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t w = pack2<BF>(s[2 * half], s[2 * half + 1]);
            hi[half] = transposed(w);
            // bf16 keeps 8 bits of a weight: what it loses goes in as a second term. fp16's 11 bits are those of the result (and see LIFT).
            if (BF) {
                const float2 u = unpack2<BF>(w);
                lo[half] = transposed(pack2<BF>(s[2 * half] - u.x, s[2 * half + 1] - u.y));
            }
        }
        const uint32_t r = (lane & 7) + ((lane >> 4) & 1) * 8;
#pragma unroll
        for (int j = 0; j < HD / 16; j++) {
            uint32_t f[4];
            ldsm4_t(f, vt + r * ROW + (((2 * j + ((lane >> 3) & 1)) ^ (r & 7)) * 16));
            mma16<BF>(o[j], f, hi[0], hi[1]);
            if (BF) mma16<BF>(o[j], f, lo[0], lo[1]);
        }
    }

    __device__ __forceinline__ void write(const SharedArgs& A, const Item& I, uint32_t lane) {
        const uint32_t g8 = lane >> 2, q4 = lane & 3;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const uint32_t r = q4 * 2 + e;
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
            if (r < I.rows) {
                if (g8 == 0) A.part_ml[I.out + r] = make_float2(m[e], l[e] * UNLIFT<BF>);
#pragma unroll
                for (int j = 0; j < HD / 8; j++) A.part_o[(I.out + r) * HD + j * 8 + g8] = o[j / 2][j % 2 * 2 + e] * UNLIFT<BF>;
            }
        }
    }
};

// RT warps share an item, 16 rows each (RT: 1, 2, 4 or 8; 0: one warp and at most 8 rows), and the tiles of 16 RT positions that they bring in by cp.async. They meet once a
// tile among themselves and with nobody else, so that what an item costs to begin and to end is other groups' time: eight warps an
// SM, 24 KB of tiles each (twelve of 16 KB where rows are at most 8). A CTA to an item, with 64 positions split over its warps, took 93 us where a group to an item
// of whatever few rows took 89 (32 sequences, tails of 1024 to 4096, before rows of at most 8 had their own form, which takes 74).
template <int HD, int RT>
__host__ __device__ constexpr int warp_stages() { return (HD == 128 ? 1 : 2) * (RT ? 3 : 2); }
template <int RT>
__host__ __device__ constexpr int warps_of() { return RT == 8 ? 8 : 4; }
template <int HD, int RT>
__host__ __device__ constexpr size_t parts_smem() { return (size_t)warps_of<RT>() * warp_stages<HD, RT>() * 64 * HD + (MAX_BATCH + 4) * 4; }

template <int RT>
__host__ __device__ constexpr int parts_ctas() { return RT == 8 ? 1 : RT ? 2 : 3; }

template <bool BF, int HD, int RT>
__global__ void __launch_bounds__(warps_of<RT>() * 32, parts_ctas<RT>()) shared_parts_kernel(const SharedArgs A, uint32_t prefix_items, uint32_t with_tails, uint32_t beside) {
    constexpr uint32_t W = RT ? RT : 1, ST = warp_stages<HD, RT>(), ROW = HD * 2, TP = 16 * W, HALF = TP * ROW, NT = warps_of<RT>() * 32, GROUPS = warps_of<RT>() / W;
    extern __shared__ __align__(128) unsigned char smem[];
    uint32_t* cum = (uint32_t*)(smem + GROUPS * ST * 2 * HALF);
    __shared__ uint32_t s_k, s_next[GROUPS][2];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, q4 = lane & 3, group = warp / W, part = warp % W;
    const uint32_t base = smem_addr(smem), ring = base + group * ST * 2 * HALF;
    auto meet = [&] {
        if (W == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(W * 32) : "memory");
    };
    // Beside the prefix's kernel, which lets this one start when all its CTAs are past their own wait. That says when, not what is visible here: the
    // prefix's token does. A CTA that does not find it waits for the prefix's end. The merge waits for this kernel alone, so this one does not
    // end before the other.
    if (!beside) pdl_wait();
    pdl_release();
    if (beside) {
        // A CTA that comes up when all items have been handed out has nothing left to work out: an earlier one left their number. The first
        // goes on all the same, since it writes the plan.
        if (threadIdx.x == 0) {
            uint64_t token;
            asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(token) : "l"(A.start) : "memory");
            const uint32_t all = *(volatile uint32_t*)(A.next + 1), out = *(volatile uint32_t*)A.next;
            s_k = token != A.token ? 2u : blockIdx.x && all && out >= all - 1 ? 1u : 0u;
        }
        __syncthreads();
        const uint32_t found = s_k;
        if (found) pdl_wait();
        if (found == 1) return;
        __syncthreads();
    }
    if (with_tails) {
        if (warp == 0) {
            const uint32_t k = cut_tails(A, cum);
            if (lane == 0) s_k = k;
        }
        __syncthreads();
        if (blockIdx.x == 0)
            for (uint32_t b = threadIdx.x; b <= A.batch; b += NT) A.plan[b] = cum[b];
    }
    const uint32_t items = prefix_items + (with_tails ? cum[A.batch] * A.kv_heads : 0), k = with_tails ? s_k : 0;
    // Beside the prefix's kernel most CTAs come up when that one leaves the SMs, and the first take what the others have not begun:
    // items are handed out by a counter.
    uint32_t w = blockIdx.x + gridDim.x * group, turn = 0;
    if (beside) {
        if (threadIdx.x == 0) *(volatile uint32_t*)(A.next + 1) = items + 1;
        if (part == 0 && lane == 0) s_next[group][1] = atomicAdd(A.next, 1u);
        meet();
        w = s_next[group][1];
    }
    for (; w < items; turn ^= 1) {
        uint32_t ahead = w + gridDim.x * GROUPS;
        if (beside && part == 0 && lane == 0) ahead = atomicAdd(A.next, 1u);
        const Item I = item_of<HD>(A, cum, k, w, prefix_items);
        const size_t pitch = 2 * I.v_off;
        const uint32_t tiles = (I.to - I.from + TP - 1) / TP, row0 = part * 16;
        auto load = [&](uint32_t i) {
            if (i < tiles) {
                const uint32_t st = ring + (i % ST) * 2 * HALF;
#pragma unroll
                for (uint32_t u = 0; u < HD / 16; u++) {
                    const uint32_t e = u * (W * 32) + part * 32 + lane, r = e / (HD / 8), ch = e % (HD / 8), pos = I.from + i * TP + r;
                    const bool in = pos < I.to;                     // rows past the end: zeros, whatever the cache holds there
                    const uint16_t* src = I.kbase + (in ? (size_t)pos * pitch + ch * 8 : 0);
                    const uint32_t dst = st + r * ROW + ((ch ^ (r & 7)) * 16);
                    cp16(dst, src, in ? 16 : 0);
                    cp16(dst + HALF, src + (in ? I.v_off : 0), in ? 16 : 0);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (uint32_t i = 0; i < ST - 1; i++) load(i);
        if constexpr (RT == 0) {
            Few<BF, HD> rows;
            rows.begin(A, I, lane);
            for (uint32_t i = 0; i < tiles; i++) {
                cp_wait<ST - 2>();
                meet();
                load(i + ST - 1);                                     // over the tile before, which all lanes have read
                const uint32_t kt = (i % ST) * 2 * HALF + (ring - base);
                rows.step(A, I, I.from + i * TP, base + kt, base + kt + HALF, smem + kt + HALF, lane);
            }
            cp_wait<0>();
            if (lane == 0) s_next[group][turn] = ahead;
            meet();                                                // the next item's tiles go over the ones just read
            w = s_next[group][turn];
            rows.write(A, I, lane);
            continue;
        }
        uint32_t qf[HD / 16][4];
        int lim[2];                                                   // the first position that a row does not see
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = row0 + g8 + half * 8;
            const bool in = r < I.rows;
            lim[half] = I.last ? min((int)I.to, (int)(I.n + r / A.rep + 1) - (int)A.q_len) : (int)I.to;
            const uint16_t* qp = A.q + (in ? (size_t)(I.token0 + r / A.rep) * A.q_stride + (size_t)(I.h * A.rep + r % A.rep) * HD : 0) + q4 * 2;
#pragma unroll
            for (int x = 0; x < HD / 16; x++) {
                qf[x][half] = in ? *(const uint32_t*)(qp + x * 16) : 0u;
                qf[x][half + 2] = in ? *(const uint32_t*)(qp + x * 16 + 8) : 0u;
            }
        }
        float o[HD / 8][4] = {};
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        for (uint32_t i = 0; i < tiles; i++) {
            cp_wait<ST - 2>();
            meet();
            load(i + ST - 1);                                         // over the tile before, which all have read
#pragma unroll 1
            for (uint32_t sub = 0; sub < RT && row0 < I.rows; sub++) {
                const uint32_t p0 = I.from + i * TP + sub * 16, kt = ring + (i % ST) * 2 * HALF + sub * 16 * ROW, vt = kt + HALF;
                if (p0 >= I.to) break;
                float s[2][4] = {};
                {
                    const uint32_t r = (lane & 7) + ((lane >> 4) & 1) * 8;
#pragma unroll
                    for (int x = 0; x < HD / 16; x++) {
                        uint32_t f[4];
                        ldsm4(f, kt + r * ROW + (((2 * x + ((lane >> 3) & 1)) ^ (r & 7)) * 16));
                        mma16<BF>(s[0], qf[x], f[0], f[1]);
                        mma16<BF>(s[1], qf[x], f[2], f[3]);
                    }
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool in = (int)(p0 + t * 8 + q4 * 2 + (e & 1)) < lim[e >> 1];
                        s[t][e] = in ? s[t][e] * A.sc : -INFINITY;
                        mx[e >> 1] = fmaxf(mx[e >> 1], s[t][e]);
                    }
                if (I.tail && A.scores) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const uint32_t r = row0 + g8 + half * 8;
                        float* sp = A.scores + (((size_t)I.b * A.kv_heads + I.h) * I.rows + r) * A.nslots;
                        if (r < I.rows)
#pragma unroll
                            for (int t = 0; t < 2; t++) {
                                const uint32_t p = p0 + t * 8 + q4 * 2;
                                if (p < I.to) sp[p] = s[t][2 * half];
                                if (p + 1 < I.to) sp[p + 1] = s[t][2 * half + 1];
                            }
                    }
                }
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
                    mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
                }
                if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const float mn = fmaxf(m[half], mx[half]), f = m[half] == -INFINITY ? 0.0f : sm100::ex2(m[half] - mn);
                        if (mn > m[half]) {
                            m[half] = mn;
                            l[half] *= f;
#pragma unroll
                            for (int j = 0; j < HD / 8; j++) { o[j][2 * half] *= f; o[j][2 * half + 1] *= f; }
                        }
                    }
                }
                const float off[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        s[t][e] = weight<BF>(s[t][e], off[e >> 1]);
                        l[e >> 1] += s[t][e];
                    }
                // Positions that only some rows see have weight 0 for the others, which is 0 times their values: where one of those is no
                // number, the tile's values are added row by row instead.
                bool odd = false;
                if (I.last && p0 + 16 > I.c && I.n > I.c) {
                    constexpr uint32_t EXP = BF ? 0x7f807f80u : 0x7c007c00u;
#pragma unroll 1
                    for (uint32_t u = 0; u < HD / 16; u++) {
                        const uint32_t e = u * 32 + lane, r = e / (HD / 8);
                        const uint4 v = *(const uint4*)(smem + (vt - base) + r * ROW + ((e % (HD / 8)) ^ (r & 7)) * 16);
                        for (uint32_t x : {v.x, v.y, v.z, v.w}) odd |= (x & EXP & 0xffffu) == (EXP & 0xffffu) || (x & EXP & 0xffff0000u) == (EXP & 0xffff0000u);
                    }
                    odd = __any_sync(0xffffffffu, odd);
                }
                if (odd) {
#pragma unroll 1
                    for (uint32_t col = 0; col < 16; col++) {
                        const int from = (int)((lane & ~3u) + (col % 8) / 2);
                        float p[2];
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            const float a = col < 8 ? s[0][2 * half] : s[1][2 * half], b = col < 8 ? s[0][2 * half + 1] : s[1][2 * half + 1];
                            p[half] = __shfl_sync(0xffffffffu, col % 2 ? b : a, from);
                        }
#pragma unroll
                        for (int j = 0; j < HD / 8; j++) {
                            const float2 v = unpack2<BF>(*(const uint32_t*)(smem + (vt - base) + col * ROW + ((j ^ (col & 7)) * 16) + q4 * 4));
#pragma unroll
                            for (int half = 0; half < 2; half++)
                                if ((int)(p0 + col) < lim[half]) { o[j][2 * half] = fmaf(p[half], v.x, o[j][2 * half]); o[j][2 * half + 1] = fmaf(p[half], v.y, o[j][2 * half + 1]); }
                        }
                    }
                    continue;
                }
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {                          // fragment register e: tile e / 2, rows of half e % 2
                    const float a = s[e >> 1][2 * (e & 1)], c2 = s[e >> 1][2 * (e & 1) + 1];
                    hi[e] = pack2<BF>(a, c2);
                    // bf16 keeps 8 bits of a weight: what it loses goes in as a second term. fp16's 11 bits are those of the result (and see LIFT).
                    if (BF) {
                        const float2 u = unpack2<BF>(hi[e]);
                        lo[e] = pack2<BF>(a - u.x, c2 - u.y);
                    }
                }
                const uint32_t r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
                for (int j = 0; j < HD / 16; j++) {
                    uint32_t f[4];
                    ldsm4_t(f, vt + r * ROW + (((2 * j + ((lane >> 4) & 1)) ^ (r & 7)) * 16));
                    mma16<BF>(o[2 * j], hi, f[0], f[1]);
                    mma16<BF>(o[2 * j + 1], hi, f[2], f[3]);
                    if (BF) {
                        mma16<BF>(o[2 * j], lo, f[0], f[1]);
                        mma16<BF>(o[2 * j + 1], lo, f[2], f[3]);
                    }
                }
            }
        }
        cp_wait<0>();
        if (part == 0 && lane == 0) s_next[group][turn] = ahead;
        meet();                                                    // the next item's tiles go over the ones just read
        w = s_next[group][turn];
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t r = row0 + g8 + half * 8;
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
            l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
            if (r < I.rows) {
                if (q4 == 0) A.part_ml[I.out + r] = make_float2(m[half], l[half] * UNLIFT<BF>);
#pragma unroll
                for (int j = 0; j < HD / 8; j++) *(float2*)&A.part_o[(I.out + r) * HD + j * 8 + q4 * 2] = make_float2(o[j][2 * half] * UNLIFT<BF>, o[j][2 * half + 1] * UNLIFT<BF>);
            }
        }
    }
    if (beside) pdl_wait();
}

// Places of a row's partial results: `first` + i * step for i < count, of the prefix and of the tail.
struct RowParts { uint32_t p_first, p_step, p_count, t_first, t_step, t_count; };

__device__ __forceinline__ RowParts row_parts(const SharedArgs& A, const uint32_t* plan, uint32_t token, uint32_t head) {
    RowParts x;
    const uint32_t h = A.by_rep(head), g = head - h * A.rep, tile = A.by_p_tokens(token), b = A.by_q_len(token), rows = A.q_len * A.rep;
    x.p_step = A.p_tokens * A.rep;
    x.p_count = A.p_slices;
    x.p_first = (tile * A.kv_heads + h) * A.p_slices * x.p_step + (token - tile * A.p_tokens) * A.rep + g;
    x.t_step = A.kv_heads * rows;
    x.t_count = x.t_first = 0;
    if (A.nslots) {
        const uint32_t c0 = plan[b];
        x.t_count = plan[b + 1] - c0;
        x.t_first = (uint32_t)A.p_rows() + (c0 * A.kv_heads + h) * rows + (token - b * A.q_len) * A.rep + g;
    }
    return x;
}
__device__ __forceinline__ size_t part_at(const RowParts& x, uint32_t i) {
    return i < x.p_count ? x.p_first + i * x.p_step : x.t_first + (i - x.p_count) * x.t_step;
}
__device__ __forceinline__ float part_factor(float2 ml, float M) { return ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : sm100::ex2(ml.x - M); }

constexpr uint32_t W_CHUNK = 1024;

// The first `weight_blocks` CTAs: 1024 tail positions of a (sequence, key head) each. The others stay and walk the rows of the result, WR warps
// to one, with eight partial results on their way at a time and maxima and sums beside them. What a call's end takes is
// latencies one behind the other: 2048 rows of 18 slices and their tails took 20 us by a warp each that read the maxima first, 10
// this way.
template <bool BF, int HD, int WR>
__global__ void __launch_bounds__(256, 3) shared_merge_kernel(const SharedArgs A, uint32_t weight_blocks, uint32_t chunks) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_release();
    if (blockIdx.x == 0 && threadIdx.x == 0) *A.start = 0;
    if (blockIdx.x >= weight_blocks) {
        __shared__ uint32_t plan[MAX_BATCH + 1];
        if (A.nslots)
            for (uint32_t b = threadIdx.x; b <= A.batch; b += 256) plan[b] = A.plan[b];
        __syncthreads();
        // a CTA's turn: 8 / WR neighbouring heads of a token
        const uint32_t heads = A.kv_heads * A.rep, wr = warp % WR, each = (heads + 8 / WR - 1) / (8 / WR), turns = A.batch * A.q_len * each;
        for (uint32_t turn = blockIdx.x - weight_blocks; turn < turns; turn += gridDim.x - weight_blocks) {
            const uint32_t token = turn / each, head = (turn - token * each) * (8 / WR) + warp / WR;
            const bool there = head < heads;
            constexpr int V = HD / 32, U = 8;
            float acc[V] = {};
            float M = -INFINITY, L = 0.0f;
            if (there) {
                const RowParts x = row_parts(A, plan, token, head);
                const uint32_t count = x.p_count + x.t_count;
                for (uint32_t i0 = wr * U; i0 < count; i0 += WR * U) {
                    float2 ml[U];
                    float v[U][V];
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        ml[u] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                        for (int e = 0; e < V; e++) v[u][e] = 0.0f;
                        if (i0 + u < count) {
                            const size_t at = part_at(x, i0 + u);
                            ml[u] = __ldcg(&A.part_ml[at]);
                            const float* p = A.part_o + at * HD + lane * V;
                            if constexpr (V == 4) { const float4 w = __ldcg((const float4*)p); v[u][0] = w.x; v[u][1] = w.y; v[u][2] = w.z; v[u][3] = w.w; }
                            else { const float2 w = __ldcg((const float2*)p); v[u][0] = w.x; v[u][1] = w.y; }
                        }
                    }
                    float top = M;
#pragma unroll
                    for (int u = 0; u < U; u++) top = fmaxf(top, ml[u].x);
                    const float back = part_factor(make_float2(M, L), top);
                    L *= back;
#pragma unroll
                    for (int e = 0; e < V; e++) acc[e] *= back;
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const float f = part_factor(ml[u], top);
                        L = fmaf(ml[u].y, f, L);
#pragma unroll
                        for (int e = 0; e < V; e++) acc[e] = fmaf(v[u][e], f, acc[e]);
                    }
                    M = top;
                }
            }
            if (WR > 1) {
                __shared__ float sums[8][HD];
                __shared__ float2 sums_ml[8];
                __syncthreads();                            // the turn before has been read
                if (lane == 0) sums_ml[warp] = make_float2(M, L);
#pragma unroll
                for (int e = 0; e < V; e++) sums[warp][e * 32 + lane] = acc[e];
                __syncthreads();
                if (wr || !there) continue;
                float top = M;
#pragma unroll
                for (int w = 1; w < WR; w++) top = fmaxf(top, sums_ml[warp + w].x);
                const float back = part_factor(make_float2(M, L), top);
                L *= back;
#pragma unroll
                for (int e = 0; e < V; e++) acc[e] *= back;
#pragma unroll
                for (int w = 1; w < WR; w++) {
                    const float f = part_factor(sums_ml[warp + w], top);
                    L = fmaf(sums_ml[warp + w].y, f, L);
#pragma unroll
                    for (int e = 0; e < V; e++) acc[e] = fmaf(sums[warp + w][e * 32 + lane], f, acc[e]);
                }
            }
            if (!there) continue;
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;      // a row that sees nothing: zeros
            uint32_t* out = (uint32_t*)(A.out + ((size_t)token * heads + head) * HD + lane * V);
            if (V == 4) *(uint2*)out = make_uint2(pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[V - 2] * inv, acc[V - 1] * inv));
            else *out = pack2<BF>(acc[0] * inv, acc[1] * inv);
        }
        return;
    }
    __shared__ float2 norm[MAX_ROWS];       // {maximum, 1 / sum} of the rows of the key head
    __shared__ int sees[MAX_ROWS];          // positions of the tail that they see: a sum that is no number is none of the others' matter
    const uint32_t u = blockIdx.x, p0 = (u % chunks) * W_CHUNK, h = (u / chunks) % A.kv_heads, b = u / chunks / A.kv_heads;
    const uint32_t n = tail_length(A, b), rows = A.q_len * A.rep;
    if (p0 >= n) return;
    const size_t head = (size_t)b * A.kv_heads + h;
    // what does not need the rows' sums is on its way before them: the scores of four rows
    float sum[4], s0[4][4];
    const float* scores = A.scores + head * rows * A.nslots + p0 + threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const bool in = p0 + i * 256 + threadIdx.x < n;
        sum[i] = in && A.weights_in ? A.weights_in[head * A.nslots + p0 + i * 256 + threadIdx.x] : 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < 4; r++) s0[r][i] = in && r < rows ? __ldcg(scores + (size_t)r * A.nslots + i * 256) : -INFINITY;
    }
    for (uint32_t r = warp; r < rows; r += 8) {
        const uint32_t t = A.by_rep(r);
        const RowParts x = row_parts(A, A.plan, b * A.q_len + t, h * A.rep + r - t * A.rep);
        const uint32_t count = x.p_count + x.t_count;
        const float2 none = make_float2(-INFINITY, 0.0f), first = lane < count ? __ldcg(&A.part_ml[part_at(x, lane)]) : none;
        float M = first.x;
        for (uint32_t i = lane + 32; i < count; i += 32) M = fmaxf(M, __ldcg(&A.part_ml[part_at(x, i)]).x);
        M = warp_max(M);
        float L = first.y * part_factor(first, M);
        for (uint32_t i = lane + 32; i < count; i += 32) {
            const float2 ml = __ldcg(&A.part_ml[part_at(x, i)]);
            L = fmaf(ml.y, part_factor(ml, M), L);
        }
        L = warp_sum(L);
        if (lane == 0) {
            norm[r] = make_float2(M == -INFINITY ? 0.0f : M, L == 0.0f ? 0.0f : 1.0f / L);
            sees[r] = (int)(n + t + 1) - (int)A.q_len;
        }
    }
    __syncthreads();
    const int p = (int)(p0 + threadIdx.x);
    float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t r = 0; r < 4; r++)
        if (r < rows) {
            const float2 x = norm[r];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (p + i * 256 < sees[r]) add[i] = fmaf(sm100::ex2(s0[r][i] - x.x), x.y, add[i]);
        }
#pragma unroll 2
    for (uint32_t r = 4; r < rows; r++) {
        const float2 x = norm[r];
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (p + i * 256 < sees[r]) add[i] = fmaf(sm100::ex2(__ldcg(scores + (size_t)r * A.nslots + i * 256) - x.x), x.y, add[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (p0 + i * 256 + threadIdx.x < n) A.weights[head * A.nslots + p0 + i * 256 + threadIdx.x] = sum[i] + add[i];
}

template <bool BF, int HD, int RT>
bool launch_parts(cudaStream_t st, const SharedArgs& a, uint32_t prefix_items, bool tails, bool beside) {
    static int have[64] = {};
    if (!ensure_dyn_smem(shared_parts_kernel<BF, HD, RT>, parts_smem<HD, RT>(), have)) return false;
    const size_t items = prefix_items + (tails ? ((size_t)a.t_slices + a.batch) * a.kv_heads : 0);
    if (!items) return true;
    g_launches++;
    return launch_pdl(shared_parts_kernel<BF, HD, RT>, dim3((uint32_t)std::min<size_t>(items, (size_t)SMS * parts_ctas<RT>())), dim3(warps_of<RT>() * 32),
                      parts_smem<HD, RT>(), st, a, prefix_items, tails ? 1u : 0u, beside ? 1u : 0u) == cudaSuccess;
}
template <bool BF, int HD>
bool launch_parts_rt(cudaStream_t st, const SharedArgs& a, uint32_t rt, uint32_t prefix_items, bool tails, bool beside) {
    switch (rt) {
        case 0: return launch_parts<BF, HD, 0>(st, a, prefix_items, tails, beside);
        case 1: return launch_parts<BF, HD, 1>(st, a, prefix_items, tails, beside);
        case 2: return launch_parts<BF, HD, 2>(st, a, prefix_items, tails, beside);
        case 4: return launch_parts<BF, HD, 4>(st, a, prefix_items, tails, beside);
        default: return launch_parts<BF, HD, 8>(st, a, prefix_items, tails, beside);
    }
}
template <bool BF, int HD>
bool launch_merge(cudaStream_t st, const SharedArgs& a) {
    const size_t tokens = (size_t)a.batch * a.q_len, heads = (size_t)a.kv_heads * a.rep;
    const uint32_t chunks = (a.nslots + W_CHUNK - 1) / W_CHUNK;
    // four warps to a row while they all find room on the SMs
    const bool wide = tokens * heads <= 16 * SMS;
    const size_t blocks = std::min<size_t>(tokens * (wide ? (heads + 1) / 2 : (heads + 7) / 8), SMS * 3), more = a.weights ? (size_t)chunks * a.batch * a.kv_heads : 0;
    g_launches++;
    return launch_pdl(wide ? shared_merge_kernel<BF, HD, 4> : shared_merge_kernel<BF, HD, 1>, dim3((uint32_t)(blocks + more)), dim3(256), 0, st, a, (uint32_t)more,
                      std::max(1u, chunks)) == cudaSuccess;
}

uint32_t row_tiles(size_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

struct Layout { size_t ml, o, scores, total; uint32_t t_rt; bool umma; };

// How a call's work is cut and where its partial results lie. false: sizes the kernels do not take.
bool lay_out(SharedArgs& a, uint32_t n_heads, uint32_t hd, bool with_weights, Layout& l, const char** why) {
    *why = "attn shared: bad shape";
    if (!a.batch || !a.q_len || !n_heads || !a.kv_heads || n_heads % a.kv_heads) return false;
    *why = "attn shared: head_dim is 64 or 128";
    if (hd != 64 && hd != 128) return false;
    a.rep = n_heads / a.kv_heads;
    *why = "attn shared: up to 1024 sequences, 16 new tokens and 128 rows (q_len * n_heads / kv_heads) to a key head, 65535 (sequence, key head) pairs";
    if (a.batch > MAX_BATCH || a.q_len > MAX_Q || (size_t)a.q_len * a.rep > MAX_ROWS || (size_t)a.batch * a.kv_heads > 65535) return false;
    *why = "attn shared: up to 2^30 prefix positions and 2^24 slots";
    if (a.n_prefix > (1u << 30) || a.nslots > (1u << 24)) return false;
    *why = "attn shared: weights of tails that have no slots";
    if (with_weights && !a.nslots) return false;
    const size_t tokens = (size_t)a.batch * a.q_len, rows = tokens * a.rep;
    const uint32_t tail_rows = a.q_len * a.rep, t_rt = row_tiles(tail_rows);
    // slices of the tails: three to a group of warps that one row tile makes, one or two where more do (64 sequences x 8 tokens: 6 an SM 165 us,
    // 12 170), 23 an SM, which has twelve warps, for rows of at most 8: the best of
    // three at one size (32 sequences with weights: 23 an SM 74.7 us, 16 78.8, 27 79.7)
    a.t_slices = std::max(1u, (tail_rows <= 8 ? 23 : t_rt == 1 ? 24 : std::max(3u, 12 / t_rt)) * SMS / a.kv_heads);
    // The prefix goes with the tails, in their launch, while its rows fit into their row tile, or are in few tiles of 16 and meet few
    // positions; else on tcgen05. 8 heads of 128, 32 rows: 512 positions 11.2 us with the tails, 13.3 on tcgen05; 2048 15.0 and
    // 14.9; 8192 24.9 and 20.1. 64 rows: 512 12.2 and 13.8; 2048 20.6 and 19.9. 128 rows: 512 13.4 and 14.4.
    l.t_rt = t_rt;
    l.umma = rows > t_rt * 16 && !(t_rt == 1 && rows * a.n_prefix <= 65536);
    a.p_tokens = (uint32_t)std::min<size_t>(tokens, (l.umma ? 128 : t_rt * 16) / a.rep);
    a.p_tiles = (uint32_t)((tokens + a.p_tokens - 1) / a.p_tokens);
    if (tail_rows <= 8 && (l.umma || rows <= 8 || !a.n_prefix)) l.t_rt = 0;
    const uint32_t unit = l.umma ? 128 : TILE, tiles = (a.n_prefix + unit - 1) / unit;
    a.p_slices = a.p_len = 0;
    if (tiles) {
        const uint32_t groups = (l.umma && a.p_tiles > 1 ? (a.p_tiles + 1) / 2 : a.p_tiles) * a.kv_heads, fit = l.umma ? SMS : SMS * (l.t_rt ? 8 / t_rt : 12);
        uint32_t best = std::min(tiles, std::max(1u, fit / groups));
        if (l.umma) {
            // What a number of slices costs, in us: a CTA takes about 7 and 2.6 a tile of two row tiles (1.6 of one). SMs that have none
            // work on the tails meanwhile, 43 KB a us each, 30 while slices are one tile; what is left of those behind the prefix begins
            // 4 us later. The tails are taken as half full. (Heads of 128; those of 64 go by the same prices, which were
            // not measured for them.) 8 sequences behind 8192 positions: 16 slices, which fill the SMs best, 32.8 us,
            // this way 26.6 (replayed, L2 cold); 64 behind 32768: 18 slices 95.4, 84.6; 32 with 2048 slots behind 16384: 67.3, 63.1.
            const bool short_ones = (size_t)a.batch * a.nslots / 2 / TILE <= a.t_slices;
            const double per = a.p_tiles > 1 ? 2.6 : 1.6, work = (double)a.batch * a.kv_heads * a.nslots * hd * 4 / 2 / (short_ones ? 30e3 : 43e3);
            double least = 1e30;
            for (uint32_t s = 1; s <= std::min(tiles, fit); s++) {
                const uint32_t ctas = groups * s, rounds = (ctas + SMS - 1) / SMS;
                const double t = rounds * (7.0 + per * ((tiles + s - 1) / s)), left = work - (rounds == 1 ? (SMS - ctas) * t : 0.0);
                const double cost = t + (left > 0.0 ? left / SMS + 4.0 : 0.0);
                if (cost < least) { least = cost; best = s; }
            }
        }
        a.p_len = (tiles + best - 1) / best * unit;
        a.p_slices = (a.n_prefix + a.p_len - 1) / a.p_len;
    }
    const size_t t_rows = a.nslots ? ((size_t)a.t_slices + a.batch) * a.kv_heads * a.q_len * a.rep : 0, parts = a.p_rows() + t_rows;
    *why = "attn shared: 2^31 partial results at most";
    if (parts >= (1ull << 31)) return false;
    a.by_rep = Div(a.rep); a.by_q_len = Div(a.q_len); a.by_p_tokens = Div(a.p_tokens);
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    l.ml = up((size_t)(a.batch + 5) * 4);                // next, start, plan
    l.o = l.ml + up(parts * 8);
    l.scores = l.o + up(parts * hd * 4);
    l.total = l.scores + (with_weights ? up((size_t)a.batch * a.kv_heads * a.q_len * a.rep * a.nslots * 4) : 0);
    return true;
}

}  // namespace

bool k_shared_parts(cudaStream_t st, const SharedArgs& a, uint32_t hd, bool bf16, uint32_t rt, bool prefix, bool tails, bool beside) {
    const uint32_t items = prefix ? a.p_tiles * a.kv_heads * a.p_slices : 0;
    if (hd == 128) return bf16 ? launch_parts_rt<true, 128>(st, a, rt, items, tails, beside) : launch_parts_rt<false, 128>(st, a, rt, items, tails, beside);
    return bf16 ? launch_parts_rt<true, 64>(st, a, rt, items, tails, beside) : launch_parts_rt<false, 64>(st, a, rt, items, tails, beside);
}
bool k_shared_merge(cudaStream_t st, const SharedArgs& a, uint32_t hd, bool bf16) {
    if (hd == 128) return bf16 ? launch_merge<true, 128>(st, a) : launch_merge<false, 128>(st, a);
    return bf16 ? launch_merge<true, 64>(st, a) : launch_merge<false, 64>(st, a);
}

// Not 0, and of 2^64 that a workspace may hold: a multiple of an odd number, from a place that the clock gives.
static uint64_t call_token() {
    static std::atomic<uint64_t> n{(uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() * 2654435761u};
    const uint64_t t = n.fetch_add(0x9e3779b97f4a7c15ull);
    return t ? t : 1;
}

bool on_this_device(const void* p, const char* what) {
    int dev = -1;
    cudaPointerAttributes at;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaPointerGetAttributes(&at, p) == cudaSuccess &&
        (at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == dev)))
        return true;
    cudaGetLastError();
    g.last_error = std::string(what) + " is no memory of the current device";
    return false;
}

}  // namespace gehtp

using namespace gehtp;

extern "C" size_t gehtp_attn_shared_workspace(uint32_t batch, uint32_t q_len, uint32_t n_heads, uint32_t kv_heads, uint32_t head_dim,
                                              uint32_t n_prefix, uint32_t nslots, int with_weights) {
    SharedArgs a{};
    a.batch = batch; a.q_len = q_len; a.kv_heads = kv_heads; a.n_prefix = n_prefix; a.nslots = nslots;
    Layout l;
    const char* why;
    if (!lay_out(a, n_heads, head_dim, with_weights != 0, l, &why)) { g.last_error = why; return 0; }
    return l.total;
}

extern "C" int gehtp_attn_shared(const void* q_dev, const void* prefix_dev, const void* tail_dev, const int32_t* n_tail_dev,
                                 const float* weights_in_dev, float* weights_dev, void* out_dev, uint32_t batch, uint32_t q_len,
                                 uint32_t n_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t q_stride, uint32_t n_prefix,
                                 uint32_t nslots, uint32_t dtype, float scale, void* workspace_dev, size_t workspace_bytes, void* stream) {
    auto fail = [](const char* m) { g.last_error = m; return -1; };
    SharedArgs a{};
    a.batch = batch; a.q_len = q_len; a.kv_heads = kv_heads; a.n_prefix = n_prefix; a.nslots = nslots;
    Layout l;
    const char* why;
    if (!lay_out(a, n_heads, head_dim, weights_dev != nullptr, l, &why)) return fail(why);
    if (dtype != GEHTP_DT_F16 && dtype != GEHTP_DT_BF16) return fail("attn shared: element type is GEHTP_DT_F16 or GEHTP_DT_BF16");
    // the kernels' scale is to the base of 2
    if (!(scale > 0.0f) || !std::isfinite(scale * 1.4426950408889634f)) return fail("attn shared: scale is a positive number below 2^127");
    if (!q_dev || !out_dev || !workspace_dev || (n_prefix && !prefix_dev) || (nslots && (!tail_dev || !n_tail_dev))) return fail("attn shared: null pointer");
    if (weights_in_dev && !weights_dev) return fail("attn shared: weights_in without weights");
    if (q_stride < (size_t)n_heads * head_dim || q_stride % 8) return fail("attn shared: q_stride is a multiple of 8, n_heads * head_dim at least");
    if ((((uintptr_t)q_dev) | ((uintptr_t)(n_prefix ? prefix_dev : nullptr)) | ((uintptr_t)(nslots ? tail_dev : nullptr)) | ((uintptr_t)out_dev)) & 15u)
        return fail("attn shared: q, prefix, tail and out lie on 16-byte boundaries");
    if ((uintptr_t)workspace_dev & 255u) return fail("attn shared: the workspace lies on a 256-byte boundary");
    if ((((uintptr_t)n_tail_dev) | ((uintptr_t)weights_in_dev) | ((uintptr_t)weights_dev)) & 3u) return fail("attn shared: n_tail and weights lie on 4-byte boundaries");
    const size_t w_bytes = (size_t)batch * kv_heads * nslots * 4;
    if (weights_in_dev && weights_in_dev != weights_dev && !apart(weights_in_dev, w_bytes, weights_dev, w_bytes)) return fail("attn shared: weights_in and weights overlap");
    if (workspace_bytes < l.total) {
        char m[128];
        std::snprintf(m, sizeof m, "attn shared: needs %zu bytes of workspace, got %zu", l.total, workspace_bytes);
        return fail(m);
    }
    if (!on_this_device(q_dev, "attn shared: q") || !on_this_device(out_dev, "attn shared: out") || !on_this_device(workspace_dev, "attn shared: workspace") ||
        (n_prefix && !on_this_device(prefix_dev, "attn shared: prefix")) ||
        (nslots && (!on_this_device(tail_dev, "attn shared: tail") || !on_this_device(n_tail_dev, "attn shared: n_tail"))) ||
        (weights_dev && !on_this_device(weights_dev, "attn shared: weights")) || (weights_in_dev && !on_this_device(weights_in_dev, "attn shared: weights_in")))
        return -1;
    // in place, weights_in is an output already
    const size_t tokens = (size_t)batch * q_len, row = (size_t)n_heads * head_dim, slot = (size_t)kv_heads * head_dim * 4;
    if (!all_apart({{out_dev, tokens * row * 2}, {weights_dev, weights_dev ? w_bytes : 0}, {workspace_dev, l.total}},
                   {{q_dev, ((tokens - 1) * q_stride + row) * 2}, {prefix_dev, n_prefix * slot}, {tail_dev, nslots * batch * slot},
                    {n_tail_dev, nslots ? (size_t)batch * 4 : 0}, {weights_in_dev, weights_in_dev != weights_dev ? w_bytes : 0}}))
        return fail("attn shared: an output or the workspace overlaps another operand");
    a.q = (const uint16_t*)q_dev; a.prefix = (const uint16_t*)prefix_dev; a.tail = (const uint16_t*)tail_dev; a.n_tail = n_tail_dev;
    a.weights_in = weights_in_dev; a.weights = weights_dev; a.out = (uint16_t*)out_dev; a.q_stride = q_stride;
    a.sc = scale * 1.4426950408889634f;
    unsigned char* ws = (unsigned char*)workspace_dev;
    a.next = (uint32_t*)ws; a.start = (uint64_t*)(ws + 8); a.plan = a.next + 4; a.token = call_token(); a.part_ml = (float2*)(ws + l.ml); a.part_o = (float*)(ws + l.o);
    a.scores = weights_dev ? (float*)(ws + l.scores) : nullptr;
    cudaStream_t st = (cudaStream_t)stream;
    const bool bf = dtype == GEHTP_DT_BF16, umma = n_prefix && l.umma;
    bool ok = true;
    if (umma) ok = k_shared_prefix_sm100(st, a, head_dim, bf);
    if (ok && (nslots || (n_prefix && !umma))) ok = k_shared_parts(st, a, head_dim, bf, l.t_rt, n_prefix && !umma, nslots != 0, umma);
    if (ok) ok = k_shared_merge(st, a, head_dim, bf);
    if (!ok) {
        const cudaError_t e = cudaGetLastError();
        return fail(e == cudaSuccess ? "attn shared: launch refused" : cudaGetErrorString(e));
    }
    return 0;
}
