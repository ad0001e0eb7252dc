// Eviction from KV caches by accumulated attention weight: a sequence whose cache holds more than `keep` positions keeps, per key head,
// its first `sinks`, its last `recent` and those of greatest weight between them (equal weights: the lower position); they move
// up in their order.
//
// select_head: the weights become whole numbers of the same order; passes over eight bits each find the smallest that stays (two or three
// of four, mostly: a pass whose digit stays as a whole is the last), then every thread lists those of its share of the positions.
// Rows move by the list. Every destination lies at or in front of its source, so a walk in ascending order moves a cache in place: a
// step's loads are complete before its stores, and later steps read behind all that earlier ones wrote. Columns of a row have nothing to
// do with one another; CTAs that share a cache in place share its columns, not its rows.
//
// evict_kernel: one launch. The CTAs of a cluster share a (sequence, key head); each makes the list for itself. Other CTAs' moves hide
// that where there are many: 64 sequences of 512 to 2048 positions cut to 1024 100 us in two launches, 90 in one; and a launch is some 2 us of the
// host's time: two sequences 13.5 -> 11.8 us call by call.
// evict_select_kernel, evict_move_kernel: lists that shared memory does not hold, and lengths replaced in place, which no CTA may write
// before all have read them. In place (rows that stay where they are do not move) 64 sequences of 512 to 2048 cut to 1024 take 79 us in one launch and 77 in
// two, two sequences 9.0 and 11.9.
#include <cstdio>
#include <algorithm>
#include "engine.h"
#include "launchers_batch.h"
#include "rows_common.cuh"

namespace gehtp {

namespace {

struct EvictArgs {
    const uint16_t* in;
    uint16_t* out;
    const float* w_in;
    float* w_out;
    const int32_t* n_in;
    int32_t *n_out, *kept, *list;          // list: [sequence][key head][keep]
    uint32_t batch, kv_heads, hd, nslots, keep, sinks, recent;
};

// Whole numbers in the order of the weights; no number counts as less than all of them.
__device__ __forceinline__ uint32_t order_of(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.0f);          // -0 and 0 are equal
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int ST = 512;
constexpr uint32_t LIST = 8192;            // positions of a list in shared memory

struct SelectShared {
    uint32_t hist[256], warps[ST / 32], digit, need, count;
};

__device__ __forceinline__ uint32_t length_of(const EvictArgs& A, uint32_t b) { return (uint32_t)min(max(A.n_in[b], 0), (int)A.nslots); }

// Exclusive sum over the CTA's threads; *total: of all
__device__ __forceinline__ uint32_t before_me(SelectShared& S, uint32_t v, uint32_t* total) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t x = v;
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    __syncthreads();
    if (lane == 31) S.warps[warp] = x;
    __syncthreads();
    uint32_t front = 0, all = 0;
#pragma unroll
    for (uint32_t i = 0; i < ST / 32; i++) { if (i == warp) front = all; all += S.warps[i]; }
    *total = all;
    return front + x - v;
}

// list: the positions of a key head that stay, in order (min(n, keep) of them). Ends with the list visible to the CTA.
__device__ void select_head(const EvictArgs& A, SelectShared& S, const float* w, uint32_t n, int32_t* list) {
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (n <= A.keep) {
        for (uint32_t i = tid; i < n; i += ST) list[i] = (int)i;
        __syncthreads();
        return;
    }
    // ---- the smallest number that stays, digit by digit, and how many that share its digits so far stay
    const uint32_t first = A.sinks, end = n - A.recent;
    uint32_t need = A.keep - A.sinks - A.recent, prefix = 0;
    int shift = 32;
    while (need && shift > 0) {
        shift -= 8;
        if (tid < 256) S.hist[tid] = 0;
        __syncthreads();
        for (uint32_t p = first + tid; p < end; p += ST) {
            const uint32_t k = order_of(w[p]);
            if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&S.hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (warp == 0) {                                   // lane l: digits 255 - 8 l and the seven below
            uint32_t c[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) { c[i] = S.hist[255 - 8 * lane - i]; sum += c[i]; }
            uint32_t upto = sum;
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= (uint32_t)o) upto += y;
            }
            uint32_t above = upto - sum;
            if (above < need && need <= upto) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (above < need && need <= above + c[i]) { S.digit = 255 - 8 * lane - i; S.need = need - above; S.count = c[i]; }
                    above += c[i];
                }
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | S.digit;
        need = S.need;
        if (S.count == need) break;                        // all that share these digits stay
    }
    // ---- who stays, in order: a run of positions to a thread
    const uint32_t per = (n + ST - 1) / ST, p0 = min(n, tid * per), p1 = min(n, p0 + per);
    const bool some = A.keep > A.sinks + A.recent;         // any of the middle stays
    uint32_t more = 0, same = 0, total;                    // that stay for certain, that share all digits looked at
    for (uint32_t p = p0; p < p1; p++) {
        if (p < first || p >= end) more++;
        else if (some) { const uint32_t k = order_of(w[p]) >> shift; more += k > prefix; same += k == prefix; }
    }
    const uint32_t equal = before_me(S, same, &total), left = equal < need ? min(same, need - equal) : 0;
    uint32_t at = before_me(S, more + left, &total), taken = 0;
    for (uint32_t p = p0; p < p1; p++) {
        bool stays = p < first || p >= end;
        if (!stays && some) {
            const uint32_t k = order_of(w[p]) >> shift;
            stays = k > prefix || (k == prefix && taken < left);
            taken += k == prefix;
        }
        if (stays) list[at++] = (int)p;
    }
    __syncthreads();
}

// Weights and old positions by the list; in place, zeros where positions left.
__device__ __forceinline__ void move_weights(const EvictArgs& A, size_t head, uint32_t n, const int32_t* list) {
    const float* w = A.w_in + head * A.nslots;
    float* wo = A.w_out + head * A.nslots;
    int32_t* kept = A.kept ? A.kept + head * A.keep : nullptr;
    const uint32_t count = min(n, A.keep);
    for (uint32_t i0 = 0; i0 < A.keep; i0 += ST) {
        const uint32_t i = i0 + threadIdx.x;
        const bool in = i < count;
        const int p = in ? list[i] : -1;
        const float x = in ? w[p] : 0.0f;
        __syncthreads();                                   // in place: all of a step has been read, and later steps read behind it
        if (in) wo[i] = x;
        if (kept && i < A.keep) kept[i] = p;
    }
    if (w == wo)
        for (uint32_t i = count + threadIdx.x; i < n; i += ST) wo[i] = 0.0f;
}

// Rows r0 .. end of the list, pieces c0 .. c0 + cols (16 bytes each) of the K or V half v; T threads, U pieces of each in flight.
template <int T, int U>
__device__ __forceinline__ void move_rows(const EvictArgs& A, uint32_t head, uint32_t v, uint32_t c0, uint32_t cols, uint32_t r0, uint32_t end, const int32_t* list) {
    const size_t width = (size_t)A.batch * A.kv_heads * A.hd, pitch = 2 * width / 8;     // a slot in 16-byte pieces
    const size_t base = (v * width + (size_t)head * A.hd) / 8 + c0;
    const uint4* in = (const uint4*)A.in + base;
    uint4* out = (uint4*)A.out + base;
    const bool in_place = A.in == A.out;
    const uint32_t step = T / cols, c = threadIdx.x % cols, r = threadIdx.x / cols;
    for (uint32_t i0 = r0; i0 < end; i0 += step * U) {
        uint4 x[U];
        uint32_t src[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t i = i0 + u * step + r;
            src[u] = i < end && r < step ? (uint32_t)list[i] : 0xFFFFFFFFu;
            if (in_place && src[u] == i) src[u] = 0xFFFFFFFFu;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (src[u] != 0xFFFFFFFFu) x[u] = in[src[u] * pitch + c];
        if (in_place) __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++)
            if (src[u] != 0xFFFFFFFFu) out[(size_t)(i0 + u * step + r) * pitch + c] = x[u];
    }
}

__global__ void __launch_bounds__(ST) evict_select_kernel(const EvictArgs A) {
    __shared__ SelectShared S;
    pdl_wait();
    pdl_release();
    const uint32_t n = length_of(A, blockIdx.x / A.kv_heads);
    int32_t* list = A.list + (size_t)blockIdx.x * A.keep;
    select_head(A, S, A.w_in + (size_t)blockIdx.x * A.nslots, n, list);
    move_weights(A, blockIdx.x, n, list);
}

constexpr int MT = 256, MU = 8;

// grid: (columns of [K | V] of a (sequence, key head) in parts of `cols` 16-byte pieces, (sequence, key head), parts of the rows)
__global__ void __launch_bounds__(MT) evict_move_kernel(const EvictArgs A, uint32_t cols, uint32_t rows_each) {
    pdl_wait();
    pdl_release();
    const uint32_t b = blockIdx.y / A.kv_heads, per = A.hd / 8 / cols, count = min(length_of(A, b), A.keep);
    // n_out may be n_in: what other CTAs then read gives the same count
    if (blockIdx.x == 0 && blockIdx.z == 0 && blockIdx.y % A.kv_heads == 0 && threadIdx.x == 0) A.n_out[b] = (int)count;
    const uint32_t r0 = blockIdx.z * rows_each;
    move_rows<MT, MU>(A, blockIdx.y, blockIdx.x / per, blockIdx.x % per * cols, cols, r0, min(count, r0 + rows_each), A.list + (size_t)blockIdx.y * A.keep);
}

// grid: (CTAs of a cluster, (sequence, key head)). In place a CTA has `cols` pieces of all rows, else all pieces of a part of the rows.
__global__ void __launch_bounds__(ST) evict_kernel(const EvictArgs A, uint32_t cols) {
    __shared__ SelectShared S;
    __shared__ int32_t list[LIST];
    pdl_wait();
    pdl_release();
    const uint32_t b = blockIdx.y / A.kv_heads, n = length_of(A, b), count = min(n, A.keep), pieces = A.hd / 8, per = pieces / cols;
    select_head(A, S, A.w_in + (size_t)blockIdx.y * A.nslots, n, list);
    if (A.w_in == A.w_out && gridDim.x > 1) {                 // all have read the weights before the first writes them
        cluster_arrive();
        cluster_wait();
    }
    if (blockIdx.x == 0) {
        if (blockIdx.y % A.kv_heads == 0 && threadIdx.x == 0) A.n_out[b] = (int)count;
        move_weights(A, blockIdx.y, n, list);
    }
    if (A.in == A.out) {
        for (uint32_t part = blockIdx.x; part < 2 * per; part += gridDim.x) move_rows<ST, 4>(A, blockIdx.y, part / per, part % per * cols, cols, 0, count, list);
    } else {
        const uint32_t r0 = (uint32_t)((uint64_t)count * blockIdx.x / gridDim.x), r1 = (uint32_t)((uint64_t)count * (blockIdx.x + 1) / gridDim.x);
        for (uint32_t v = 0; v < 2; v++) move_rows<ST, 4>(A, blockIdx.y, v, 0, pieces, r0, r1, list);
    }
}

const char* evict_refuses(uint32_t batch, uint32_t kv_heads, uint32_t hd, uint32_t nslots, uint32_t keep, uint32_t sinks, uint32_t recent) {
    if (!batch || !kv_heads || (size_t)batch * kv_heads > 65535) return "kv evict: 1 to 65535 (sequence, key head) pairs";
    if (!hd || hd % 8 || hd > 512) return "kv evict: head_dim is a multiple of 8, up to 512";
    if (!nslots || nslots > (1u << 24)) return "kv evict: 1 to 2^24 slots";
    if (!keep || keep > nslots) return "kv evict: keep is 1 to nslots";
    if ((size_t)sinks + recent > keep) return "kv evict: sinks and recent together are no more than keep";
    return nullptr;
}

}  // namespace

bool k_kv_evict(cudaStream_t st, const EvictArgs& a) {
    if (a.n_in != a.n_out && a.keep <= LIST) {
        // CTAs to a cluster: up to eight, while they do not fill the SMs twice
        const uint32_t heads = a.batch * a.kv_heads, pieces = a.hd / 8;
        uint32_t parts = 1, cols = pieces;
        while (parts < 8 && heads * parts * 2 <= 2 * 148) parts *= 2;
        if (a.in == a.out)
            while (cols % 2 == 0 && cols > 2 && 2 * (pieces / cols) < parts) cols /= 2;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(parts, heads); cfg.blockDim = dim3(ST); cfg.stream = st;
        g_launches++;
        return launch_pdl_cluster(evict_kernel, cfg, dim3(parts, 1, 1), a, cols) == cudaSuccess;
    }
    g_launches += 2;
    if (launch_pdl(evict_select_kernel, dim3(a.batch * a.kv_heads), dim3(ST), 0, st, a) != cudaSuccess) return false;
    // 16-byte pieces of a row half to a CTA: all of them, fewer where a cache that is moved in place would leave SMs idle
    const uint32_t pieces = a.hd / 8, heads = a.batch * a.kv_heads;
    uint32_t cols = pieces;
    if (a.in == a.out)
        while (cols % 2 == 0 && cols > 2 && heads * 2 * (pieces / cols) < 2 * 148) cols /= 2;
    const uint32_t parts = 2 * (pieces / cols), step = MT / cols * MU;
    uint32_t rows_each = a.keep, splits = 1;
    if (a.in != a.out) {
        splits = std::min((a.keep + step - 1) / step, std::max(1u, 8 * 148 / (heads * parts)));
        rows_each = (a.keep + splits - 1) / splits;
    }
    return launch_pdl(evict_move_kernel, dim3(parts, heads, splits), dim3(MT), 0, st, a, cols, rows_each) == cudaSuccess;
}

}  // namespace gehtp

using namespace gehtp;

extern "C" size_t gehtp_kv_evict_workspace(uint32_t batch, uint32_t kv_heads, uint32_t head_dim, uint32_t nslots, uint32_t keep,
                                           uint32_t sinks, uint32_t recent) {
    if (const char* why = evict_refuses(batch, kv_heads, head_dim, nslots, keep, sinks, recent)) { g.last_error = why; return 0; }
    return ((size_t)batch * kv_heads * keep * 4 + 255) / 256 * 256;
}

extern "C" int gehtp_kv_evict(const void* ring_dev, void* ring_out_dev, const float* weights_dev, float* weights_out_dev,
                              const int32_t* n_dev, int32_t* n_out_dev, int32_t* kept_dev, uint32_t batch, uint32_t kv_heads,
                              uint32_t head_dim, uint32_t nslots, uint32_t keep, uint32_t sinks, uint32_t recent,
                              void* workspace_dev, size_t workspace_bytes, void* stream) {
    auto fail = [](const char* m) { g.last_error = m; return -1; };
    if (const char* why = evict_refuses(batch, kv_heads, head_dim, nslots, keep, sinks, recent)) return fail(why);
    if (!ring_dev || !ring_out_dev || !weights_dev || !weights_out_dev || !n_dev || !n_out_dev || !workspace_dev) return fail("kv evict: null pointer");
    if ((((uintptr_t)ring_dev) | ((uintptr_t)ring_out_dev)) & 15u) return fail("kv evict: caches lie on 16-byte boundaries");
    if ((((uintptr_t)weights_dev) | ((uintptr_t)weights_out_dev) | ((uintptr_t)n_dev) | ((uintptr_t)n_out_dev) | ((uintptr_t)kept_dev)) & 3u)
        return fail("kv evict: weights, counts and kept lie on 4-byte boundaries");
    if ((uintptr_t)workspace_dev & 255u) return fail("kv evict: the workspace lies on a 256-byte boundary");
    const size_t heads = (size_t)batch * kv_heads, need = gehtp_kv_evict_workspace(batch, kv_heads, head_dim, nslots, keep, sinks, recent);
    if (ring_dev != ring_out_dev && !apart(ring_dev, heads * nslots * head_dim * 4, ring_out_dev, heads * nslots * head_dim * 4)) return fail("kv evict: ring and ring_out overlap");
    if (weights_dev != weights_out_dev && !apart(weights_dev, heads * nslots * 4, weights_out_dev, heads * nslots * 4)) return fail("kv evict: weights and weights_out overlap");
    if (n_dev != n_out_dev && !apart(n_dev, (size_t)batch * 4, n_out_dev, (size_t)batch * 4)) return fail("kv evict: n and n_out overlap");
    if (workspace_bytes < need) {
        char m[128];
        std::snprintf(m, sizeof m, "kv evict: needs %zu bytes of workspace, got %zu", need, workspace_bytes);
        return fail(m);
    }
    if (!on_this_device(ring_dev, "kv evict: ring") || !on_this_device(ring_out_dev, "kv evict: ring_out") || !on_this_device(weights_dev, "kv evict: weights") ||
        !on_this_device(weights_out_dev, "kv evict: weights_out") || !on_this_device(n_dev, "kv evict: n") || !on_this_device(n_out_dev, "kv evict: n_out") ||
        !on_this_device(workspace_dev, "kv evict: workspace") || (kept_dev && !on_this_device(kept_dev, "kv evict: kept")))
        return -1;
    const size_t ring = heads * nslots * head_dim * 4, w = heads * nslots * 4, n = (size_t)batch * 4;
    if (!all_apart({{ring_out_dev, ring}, {weights_out_dev, w}, {n_out_dev, n}, {kept_dev, kept_dev ? heads * keep * 4 : 0}, {workspace_dev, need}},
                   {{ring_dev, ring_dev != ring_out_dev ? ring : 0}, {weights_dev, weights_dev != weights_out_dev ? w : 0}, {n_dev, n_dev != n_out_dev ? n : 0}}))
        return fail("kv evict: an output or the workspace overlaps another operand");
    EvictArgs a{(const uint16_t*)ring_dev, (uint16_t*)ring_out_dev, weights_dev, weights_out_dev, n_dev, n_out_dev, kept_dev, (int32_t*)workspace_dev,
                batch, kv_heads, head_dim, nslots, keep, sinks, recent};
    if (!k_kv_evict((cudaStream_t)stream, a)) {
        const cudaError_t e = cudaGetLastError();
        return fail(e == cudaSuccess ? "kv evict: launch refused" : cudaGetErrorString(e));
    }
    return 0;
}
