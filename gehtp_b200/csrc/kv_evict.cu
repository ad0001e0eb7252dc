// Eviction from KV caches by accumulated attention weight: a sequence whose cache holds more than `keep` positions keeps, per key head,
// its first `sinks`, its last `recent` and those of greatest weight between them (equal weights: the lower position); they move
// up in their order.
//
// evict_select_kernel: a CTA per (sequence, key head). The weights become whole numbers of the same order, four passes over eight bits
// each find the smallest that stays, one pass in order writes the list of the positions that stay and moves the weights.
// evict_move_kernel: rows by the list. Every destination lies at or in front of its source, so a walk in ascending order moves a cache in
// place: a step's loads are complete before its stores, and later steps read behind all that earlier ones wrote. Columns of a row
// have nothing to do with one another; CTAs that share a cache in place share its columns, not its rows.
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

__global__ void __launch_bounds__(ST) evict_select_kernel(const EvictArgs A) {
    __shared__ uint32_t hist[256], warps[ST / 32], s_digit, s_need;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_release();
    const uint32_t b = blockIdx.x / A.kv_heads;
    const size_t head = blockIdx.x;
    const uint32_t n = (uint32_t)min(max(A.n_in[b], 0), (int)A.nslots), count = min(n, A.keep);
    const float* w = A.w_in + head * A.nslots;
    float* wo = A.w_out + head * A.nslots;
    int32_t *list = A.list + head * A.keep, *kept = A.kept ? A.kept + head * A.keep : nullptr;
    if (kept)
        for (uint32_t i = count + tid; i < A.keep; i += ST) kept[i] = -1;
    if (n <= A.keep) {
        for (uint32_t i = tid; i < n; i += ST) {
            list[i] = (int)i;
            if (kept) kept[i] = (int)i;
            if (w != wo) wo[i] = w[i];
        }
        return;
    }
    // ---- the smallest number that stays, digit by digit, and how many that are equal to it stay
    const uint32_t first = A.sinks, end = n - A.recent;
    uint32_t need = A.keep - A.sinks - A.recent, prefix = 0;
    if (need) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (uint32_t i = tid; i < 256; i += ST) hist[i] = 0;
            __syncthreads();
            for (uint32_t p = first + tid; p < end; p += ST) {
                const uint32_t k = order_of(w[p]);
                if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
            }
            __syncthreads();
            if (warp == 0) {                               // lane l: digits 255 - 8 l and the seven below
                uint32_t c[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) { c[i] = hist[255 - 8 * lane - i]; sum += c[i]; }
                uint32_t upto = sum;
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= (uint32_t)o) upto += y;
                }
                uint32_t above = upto - sum;
                if (above < need && need <= upto) {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        if (above < need && need <= above + c[i]) { s_digit = 255 - 8 * lane - i; s_need = need - above; }
                        above += c[i];
                    }
                }
            }
            __syncthreads();
            prefix = (prefix << 8) | s_digit;
            need = s_need;
        }
    } else {
        prefix = 0xFFFFFFFFu;                              // no weight's number: none of the middle stays
    }
    // ---- in order: who stays, and where it goes. equal: how many equal to `prefix` lie in front
    uint32_t placed = 0, equal = 0;
    for (uint32_t p0 = 0; p0 < n; p0 += ST) {
        const uint32_t p = p0 + tid;
        float x = 0.0f;
        bool stay = false, same = false;
        if (p < n) {
            x = w[p];
            if (p < first || p >= end) stay = true;
            else { const uint32_t k = order_of(x); stay = k > prefix; same = k == prefix && need; }
        }
        const uint32_t below = (1u << lane) - 1u, sb = __ballot_sync(0xffffffffu, same);
        if (lane == 0) warps[warp] = __popc(sb);
        __syncthreads();
        uint32_t e = equal, all = 0;
        for (uint32_t i = 0; i < ST / 32; i++) { if (i < warp) e += warps[i]; all += warps[i]; }
        equal += all;
        if (same && e + __popc(sb & below) < need) stay = true;
        const uint32_t tb = __ballot_sync(0xffffffffu, stay);
        __syncthreads();
        if (lane == 0) warps[warp] = __popc(tb);
        __syncthreads();
        uint32_t at = placed;
        all = 0;
        for (uint32_t i = 0; i < ST / 32; i++) { if (i < warp) at += warps[i]; all += warps[i]; }
        placed += all;
        at += __popc(tb & below);
        if (stay) {                                        // in place: `at` <= p, and all weights up to p0 + ST - 1 have been read
            list[at] = (int)p;
            if (kept) kept[at] = (int)p;
            wo[at] = x;
        }
        __syncthreads();
    }
    if (w == wo)
        for (uint32_t p = A.keep + tid; p < n; p += ST) wo[p] = 0.0f;
}

constexpr int MT = 256, MU = 8;

// grid: (columns of [K | V] of a (sequence, key head) in parts of `cols` 16-byte pieces, (sequence, key head), parts of the rows)
__global__ void __launch_bounds__(MT) evict_move_kernel(const EvictArgs A, uint32_t cols, uint32_t rows_each) {
    pdl_wait();
    pdl_release();
    const uint32_t b = blockIdx.y / A.kv_heads, per = A.hd / 8 / cols;
    const uint32_t n = (uint32_t)min(max(A.n_in[b], 0), (int)A.nslots), count = min(n, A.keep);
    // n_out may be n_in: what other CTAs then read gives the same count
    if (blockIdx.x == 0 && blockIdx.z == 0 && blockIdx.y % A.kv_heads == 0 && threadIdx.x == 0) A.n_out[b] = (int)count;
    const uint32_t v = blockIdx.x / per, c0 = (blockIdx.x % per) * cols;
    const size_t width = (size_t)A.batch * A.kv_heads * A.hd, pitch = 2 * width / 8;     // a slot in 16-byte pieces
    const size_t base = (v * width + (size_t)blockIdx.y * A.hd) / 8 + c0;
    const uint4* in = (const uint4*)A.in + base;
    uint4* out = (uint4*)A.out + base;
    const int32_t* list = A.list + (size_t)blockIdx.y * A.keep;
    const bool in_place = A.in == A.out;
    const uint32_t r0 = blockIdx.z * rows_each, end = min(count, r0 + rows_each), step = MT / cols;
    const uint32_t c = threadIdx.x % cols, r = threadIdx.x / cols;
    for (uint32_t i0 = r0; i0 < end; i0 += step * MU) {
        uint4 x[MU];
        uint32_t src[MU];
#pragma unroll
        for (int u = 0; u < MU; u++) {
            const uint32_t i = i0 + u * step + r;
            src[u] = i < end && r < step ? (uint32_t)list[i] : 0xFFFFFFFFu;
            if (in_place && src[u] == i) src[u] = 0xFFFFFFFFu;
        }
#pragma unroll
        for (int u = 0; u < MU; u++)
            if (src[u] != 0xFFFFFFFFu) x[u] = in[src[u] * pitch + c];
        if (in_place) __syncthreads();
#pragma unroll
        for (int u = 0; u < MU; u++)
            if (src[u] != 0xFFFFFFFFu) out[(size_t)(i0 + u * step + r) * pitch + c] = x[u];
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

bool apart(const void* a, const void* b, size_t bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x + bytes <= y || y + bytes <= x;
}

}  // namespace

bool k_kv_evict(cudaStream_t st, const EvictArgs& a) {
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
    if (ring_dev != ring_out_dev && !apart(ring_dev, ring_out_dev, heads * nslots * head_dim * 4)) return fail("kv evict: ring and ring_out overlap");
    if (weights_dev != weights_out_dev && !apart(weights_dev, weights_out_dev, heads * nslots * 4)) return fail("kv evict: weights and weights_out overlap");
    if (n_dev != n_out_dev && !apart(n_dev, n_out_dev, (size_t)batch * 4)) return fail("kv evict: n and n_out overlap");
    if (workspace_bytes < need) {
        char m[128];
        std::snprintf(m, sizeof m, "kv evict: needs %zu bytes of workspace, got %zu", need, workspace_bytes);
        return fail(m);
    }
    if (!on_this_device(ring_dev, "kv evict: ring") || !on_this_device(ring_out_dev, "kv evict: ring_out") || !on_this_device(weights_dev, "kv evict: weights") ||
        !on_this_device(weights_out_dev, "kv evict: weights_out") || !on_this_device(n_dev, "kv evict: n") || !on_this_device(n_out_dev, "kv evict: n_out") ||
        !on_this_device(workspace_dev, "kv evict: workspace") || (kept_dev && !on_this_device(kept_dev, "kv evict: kept")))
        return -1;
    EvictArgs a{(const uint16_t*)ring_dev, (uint16_t*)ring_out_dev, weights_dev, weights_out_dev, n_dev, n_out_dev, kept_dev, (int32_t*)workspace_dev,
                batch, kv_heads, head_dim, nslots, keep, sinks, recent};
    if (!k_kv_evict((cudaStream_t)stream, a)) {
        const cudaError_t e = cudaGetLastError();
        return fail(e == cudaSuccess ? "kv evict: launch refused" : cudaGetErrorString(e));
    }
    return 0;
}
