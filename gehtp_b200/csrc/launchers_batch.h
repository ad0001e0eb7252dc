// Operators for a batch of sequences that go on from one prompt (shared_attn.cu, shared_attn_sm100.cu, kv_evict.cu,
// verify_drafts.cu). All memory is the caller's: nothing is allocated, kept or remembered between calls.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <initializer_list>

namespace gehtp {

// n / d by a product, for n * d < 2^32
struct Div {
    uint64_t m;
    Div() = default;
    explicit Div(uint32_t d) : m(((1ull << 32) + d - 1) / d) {}
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return (uint32_t)((n * m) >> 32); }
};

// Attention over a shared prefix and own tails. A row is one query head of one token; the rows that meet a key head's
// prefix together are those of p_tokens tokens (a row tile), those that meet a tail are the q_len * rep of its sequence.
// Every (row tile, key head, slice of the prefix) and every (sequence, key head, slice of its tail) leaves a partial result per
// row: the sum of 2^(s - m) v, the sum of 2^(s - m) and the reference m, with s = log2(e) * scale * q.k. m is a maximum, or what the prefix's
// kernel took in its place.
struct SharedArgs {
    const uint16_t *q, *prefix, *tail;
    const int32_t* n_tail;
    const float* weights_in;
    float* weights;
    uint16_t* out;
    uint32_t batch, q_len, rep, kv_heads, n_prefix, nslots;
    size_t q_stride;
    uint32_t p_tokens, p_tiles, p_slices, p_len;   // prefix: slices of p_len positions
    uint32_t t_slices;                             // the tails of all sequences are cut into about so many slices
    Div by_rep, by_q_len, by_p_tokens;             // of heads below 2^23 by up to 128, of tokens below 2^14 by up to 16 and 128
    float sc;                                      // log2(e) * scale
    float* part_o;                                 // [partial row][head_dim], the prefix's first
    float2* part_ml;                               // [partial row] {m, sum}
    float* scores;                                 // s of every tail position: [sequence][key head][row][nslots], or NULL
    uint32_t* next;                                // where the tails' kernel runs beside the prefix's, which sets both to 0: items handed out; items + 1
    // Where it does: the prefix's kernel writes `token`, another one for every call, to *start when all in front of the call has been waited for and
    // `next` is set. Who reads it there (acquire) sees all of that too. The merge takes it away again.
    uint64_t *start, token;
    uint32_t* plan;                                // written by the first kernel: slices in front of each sequence's, batch + 1 of them
    __host__ __device__ size_t p_rows() const { return (size_t)p_tiles * kv_heads * p_slices * p_tokens * rep; }
};

// false: launch failed
bool k_shared_prefix_sm100(cudaStream_t st, const SharedArgs& a, uint32_t hd, bool bf16);
// beside: behind the prefix's kernel in the stream, at the same time as it
bool k_shared_parts(cudaStream_t st, const SharedArgs& a, uint32_t hd, bool bf16, uint32_t row_tiles, bool prefix, bool tails, bool beside);
bool k_shared_merge(cudaStream_t st, const SharedArgs& a, uint32_t hd, bool bf16);

inline bool apart(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return !a || !b || x + a_bytes <= y || y + b_bytes <= x;
}
// Operands of a call: none of `outs` may share memory with another of them or with one of `ins`. What takes no bytes shares none.
struct Span { const void* p; size_t bytes; };
inline bool apart(Span a, Span b) { return !a.bytes || !b.bytes || apart(a.p, a.bytes, b.p, b.bytes); }
inline bool all_apart(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
    for (auto o = outs.begin(); o != outs.end(); o++) {
        for (auto x = o + 1; x != outs.end(); x++)
            if (!apart(*o, *x)) return false;
        for (Span i : ins)
            if (!apart(*o, i)) return false;
    }
    return true;
}
// true: `p` is memory of the current device (or managed); else g.last_error says which argument is not
bool on_this_device(const void* p, const char* what);

}  // namespace gehtp
