// What the kernels over a paged cache share: where a token's row lies, which sequence a new token belongs to, and the checks of
// the descriptors that the host can make.
#pragma once
#include "q4_common.cuh"
#include "runtime.h"

namespace tessl {
namespace paged {

/// Two f32 -> a bf16 pair, to nearest even.
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

/// The cache as the kernels address it; strides in elements.
struct Cache {
    uint16_t *k, *v;
    uint64_t page_stride;
    uint32_t token_stride, head_stride;
    uint32_t num_pages, page_size, n_kv_heads, head_dim;
};

struct Seqs {
    const int32_t *table, *lens, *starts;  // starts may be null: one new token each
    uint32_t num_seqs, max_pages, total_new;
    uint64_t capacity;  // tokens that a row of the table has room for
};

/// A word that every block reads, through L1 (from L2, some thousand warps wait for one another at the few lines that hold
/// such words), and after the wait for the launch in front (see dev::ld_after_wait16).
__device__ __forceinline__ int32_t ld_shared_word(const int32_t *p)
{
    int32_t v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

/// Offsets and lengths come from device memory: whatever they hold, what is made of them stays inside the call's tokens and the
/// table's row.
__device__ __forceinline__ uint32_t start_of(const Seqs &q, uint32_t s)
{
    if (!q.starts) return s;
    return (uint32_t)min(max(ld_shared_word(q.starts + s), 0), (int32_t)min(q.total_new, 0x7fffffffu));
}
/// Tokens of a sequence by its length; those past q.capacity have no slot.
__device__ __forceinline__ uint32_t len_of(const Seqs &q, uint32_t s) { return (uint32_t)max(ld_shared_word(q.lens + s), 0); }

/// The sequence whose new tokens hold `row`, found by a converged warp, 32 offsets at a time; num_seqs if there is none.
__device__ __forceinline__ uint32_t seq_of_row(const Seqs &q, uint32_t row)
{
    const uint32_t lane = threadIdx.x & 31;
    if (!q.starts) return row < q.num_seqs ? row : q.num_seqs;
    // invariant: the sequence wanted, if any, is the last one with start <= row among [lo, hi)
    uint32_t lo = 0, hi = q.num_seqs;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t below = __popc(__ballot_sync(0xffffffffu, at < hi && start_of(q, at) <= row));
        if (below == 0) return q.num_seqs;
        lo += (below - 1) * step;
        hi = min(hi, lo + step);
    }
    if (hi == lo || start_of(q, lo) > row || start_of(q, lo + 1) <= row) return q.num_seqs;
    return lo;
}

/// A cache's sizes; its buffers may be missing yet.
inline Result cache_sizes_validate(const TesslPagedKv &c, const char *what)
{
    if (c.layout != TESSL_KV_TOKEN_MAJOR && c.layout != TESSL_KV_HEAD_MAJOR) return fmt("%s: unknown cache layout %u", what, c.layout);
    if (c.head_dim == 0 || c.head_dim % 8 != 0 || c.head_dim > 256)
        return fmt("%s: head_dim %u is not a multiple of 8 up to 256", what, c.head_dim);
    if (c.n_kv_heads == 0 || c.n_kv_heads > 65535) return fmt("%s: n_kv_heads %u is outside 1 .. 65535", what, c.n_kv_heads);
    if (c.page_size == 0) return fmt("%s: page_size must be non-zero", what);
    const uint64_t page = elems(c.n_kv_heads, c.head_dim) * c.page_size;  // a row < 2^24
    if (page > 0x7fffffffull) return fmt("%s: a page of %llu values is too large", what, (unsigned long long)page);
    if (c.num_pages > 0x7fffffffu) return fmt("%s: num_pages %u does not fit an int32 page id", what, c.num_pages);
    return ok();
}

inline Result cache_validate(const TesslPagedKv &c, const char *what, Cache *out)
{
    TESSL_TRY(cache_sizes_validate(c, what));
    const uint64_t row = elems(c.n_kv_heads, c.head_dim), page = row * c.page_size;
    const uint64_t need = page * c.num_pages;  // < 2^62
    TESSL_TRY(require(c.k, need, 2, What(what) + " cache k"));
    TESSL_TRY(require(c.v, need, 2, What(what) + " cache v"));
    TESSL_TRY(require_aligned16(c.k, What(what) + " cache k"));
    TESSL_TRY(require_aligned16(c.v, What(what) + " cache v"));
    const bool by_token = c.layout == TESSL_KV_TOKEN_MAJOR;
    *out = Cache{static_cast<uint16_t *>(c.k.ptr), static_cast<uint16_t *>(c.v.ptr), page,
                 by_token ? (uint32_t)row : c.head_dim, by_token ? c.head_dim : c.head_dim * c.page_size,
                 c.num_pages, c.page_size, c.n_kv_heads, c.head_dim};
    return ok();
}

inline Result seqs_sizes_validate(const TesslPagedSeqs &s, uint32_t total_new, const char *what)
{
    if (s.num_seqs > 0x7fffffffu || total_new > 0x7fffffffu)
        return fmt("%s: %u sequences, %u new tokens: more than an int32 offset counts", what, s.num_seqs, total_new);
    return ok();
}

inline Result seqs_validate(const TesslPagedSeqs &s, const TesslPagedKv &c, uint32_t total_new, const char *what, Seqs *out)
{
    TESSL_TRY(seqs_sizes_validate(s, total_new, what));
    TESSL_TRY(require(s.page_table, elems(s.num_seqs, s.max_pages), 4, What(what) + " page_table"));
    TESSL_TRY(require(s.kv_lens, s.num_seqs, 4, What(what) + " kv_lens"));
    if (s.q_starts.ptr) {
        TESSL_TRY(require(s.q_starts, (uint64_t)s.num_seqs + 1, 4, What(what) + " q_starts"));
    } else if (total_new != s.num_seqs) {
        return fmt("%s: without q_starts each sequence has one new token, but there are %u for %u sequences", what, total_new, s.num_seqs);
    }
    for (const TesslBuf *b : {&s.page_table, &s.kv_lens, &s.q_starts})
        if (((uintptr_t)b->ptr & 3u) != 0) return fmt("%s: page_table, kv_lens and q_starts must be 4-byte aligned", what);
    *out = Seqs{static_cast<const int32_t *>(s.page_table.ptr), static_cast<const int32_t *>(s.kv_lens.ptr),
                static_cast<const int32_t *>(s.q_starts.ptr), s.num_seqs, s.max_pages, total_new,
                elems(s.max_pages, c.page_size)};
    return ok();
}

/// Rows of `width` values, `stride` apart (0 = one behind the other): the stride, after a check of the buffer's reach.
inline Result rows_validate(const TesslBuf &b, uint32_t rows, uint64_t width, uint32_t *stride, size_t elem, const char *what, const char *name)
{
    if (*stride == 0) {
        if (width > 0xffffffffull) return fmt("%s: rows of %s are too long", what, name);
        *stride = (uint32_t)width;
    }
    if (*stride < width) return fmt("%s: rows of %s are %llu values long but %u apart", what, name, (unsigned long long)width, *stride);
    TESSL_TRY(require(b, rows ? (uint64_t)(rows - 1) * *stride + width : 0, elem, What(what) + " " + name));
    if (((uintptr_t)b.ptr & (elem - 1)) != 0) return fmt("%s: %s is not aligned to its elements", what, name);
    return ok();
}

}  // namespace paged
}  // namespace tessl
