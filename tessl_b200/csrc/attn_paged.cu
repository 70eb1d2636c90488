// Attention over a paged cache: checks, routes and launches.
#include <algorithm>
#include <cmath>
#include <random>
#include <type_traits>

#include "attn_paged_split.cuh"
#include "attn_paged_tile.cuh"
#include "tensormap.h"

namespace tessl {
namespace {

using attn::Params;

uint32_t padded_dim(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

/// f(std::integral_constant<int, DP>) for the padded width of a head.
template <typename F>
auto with_dim(uint32_t head_dim, F f)
{
    switch (padded_dim(head_dim)) {
    case 64: return f(std::integral_constant<int, 64>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 192: return f(std::integral_constant<int, 192>{});
    default: return f(std::integral_constant<int, 256>{});
    }
}

/// Tokens per TMA box, of those that a step or tile of keys has: a power of two that divides a page; fewer than eight would break the
/// swizzle's groups of eight rows.
uint32_t box_of(uint32_t page_size, uint32_t most) { return std::min(page_size & (0u - page_size), most); }

/// Whether the new tokens are given by offsets. A query of the workspace may come before there are any: without them a call has a new
/// token for each sequence.
bool with_starts(const TesslPagedSeqs &seqs, uint32_t total_new) { return seqs.q_starts.ptr || total_new != seqs.num_seqs; }

/// Whether a call of so many new tokens or fewer, of so many sequences or fewer, may go to the tensor-core tiles: all tokens may be of one.
bool may_want_tiles(const TesslPagedKv &cache, const TesslPagedSeqs &seqs, uint32_t total_new, uint32_t group)
{
    return with_starts(seqs, total_new) && cache.num_pages > 0 && cache.page_size % 8 == 0 && elems(total_new, group) > 32;
}

/// Whether a call of these sizes goes to the tensor-core tiles: more than 32 rows for each key head of a sequence, on average. Eight
/// sequences of up to 8000 keys, 32 heads of 128 on 8, with the kernel for few rows and with the tiles: 16 rows 56 and 60 us, 24 rows 66 and
/// 60 us, 48 rows 83 and 61 us; one sequence: 32 rows 25 and 29 us, 64 rows 42 and 39 us; four sequences of wide heads: 32 rows 51 and 50 us.
/// Those are sequences of alike numbers of rows. A chunk among many single tokens goes by the mean with them, and reads its keys once per 16
/// rows: a chunk of 256 over 30000 keys beside 63 tokens over up to 30000 takes 1735 us, a call for the chunk and one for the tokens 836;
/// of 512 over 33000 beside 255 over up to 4000 2957 and 747 us. The other way round a token has a tile of 256 rows to itself, which costs
/// less: a prompt of 4096 beside 7 tokens 275 us, in two calls 311. Sequences without new tokens lower the mean too.
bool wants_tiles(const TesslPagedKv &cache, const TesslPagedSeqs &seqs, uint32_t total_new, uint32_t group)
{
    return may_want_tiles(cache, seqs, total_new, group) && elems(total_new, group) > 32ull * seqs.num_seqs;
}

/// Blocks of the split kernel on an SM: two, of half the warps each, where there are more items than SMs, so that one reads while the other
/// starts or ends an item. With one and with two, heads as above, a token each: 64 sequences of up to 1000 keys 58 and 49 us, 24 of up to
/// 6000 keys 87 and 80 us, 12 of up to 6000 keys 51 and 50 us, 8 of up to 500 keys 11 and 16 us, one of 130001 keys 103 and 107 us.
uint32_t split_blocks(const TesslRuntime *rt, const TesslPagedKv &cache, const TesslPagedSeqs &seqs)
{
    return elems(seqs.num_seqs, cache.n_kv_heads) > (uint64_t)rt->sm_count ? 2 : 1;
}

/// Whether a call whose sequences are as long as their rows of the page table has more units than the kernels count, in 32 bits: what they
/// count are the blocks of rows and the units of keys of the route that the call takes.
bool too_much(const TesslPagedKv &cache, const TesslPagedSeqs &seqs, uint32_t total_new, uint32_t group, bool tiles)
{
    const double rows = tiles ? with_dim(cache.head_dim, [](auto dp) { return (double)attn::TileCfg<decltype(dp)::value>::ROWS; }) : attn::kSplitRows;
    const double blocks = (double)elems(total_new, group) / rows + seqs.num_seqs;
    const double most = (double)std::min<uint64_t>(elems(seqs.max_pages, cache.page_size), 0x7fffffffu) / (tiles ? attn::kTileKeys : attn::kSplitUnit) + 1;
    return blocks * most * cache.n_kv_heads >= 4294967296.0;
}

uint64_t workspace_of(const TesslRuntime *rt, const TesslPagedKv &cache, const TesslPagedSeqs &seqs, bool tiles)
{
    return with_dim(cache.head_dim, [&](auto dp) -> uint64_t {
        constexpr int DP = decltype(dp)::value;
        const uint64_t few = attn::Part<attn::kSplitRows, DP>::bytes((uint64_t)rt->sm_count * split_blocks(rt, cache, seqs));
        const uint64_t many = attn::Part<attn::TileCfg<DP>::ROWS, DP>::bytes(rt->sm_count);
        return tiles ? std::max(few, many) : few;
    });
}

/// The cache's maps for boxes of 64 columns of one key head and `box` tokens of one page.
Result cache_maps(TesslRuntime *rt, const char *what, const paged::Cache &c, uint32_t box, CUtensorMap *k, CUtensorMap *v)
{
    EncodeTiled enc;
    TESSL_TRY(tensormap_encoder(rt, what, &enc));
    const cuuint64_t dims[4] = {c.head_dim, c.n_kv_heads, c.page_size, c.num_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.head_stride * 2, (cuuint64_t)c.token_stride * 2, c.page_stride * 2};
    const cuuint32_t boxes[4] = {64, 1, box, 1};
    TESSL_TRY(make_map(enc, what, k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.k, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_128B));
    return make_map(enc, what, v, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, c.v, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <int DP, int BLOCKS>
Result launch_split(TesslRuntime *rt, const Params &p)
{
    using C = attn::SplitCfg<DP, BLOCKS>;
    const char *what = "attn_paged launch";
    attn::SplitParams sp{p, box_of(p.cache.page_size, attn::kStep)};
    sp.p.parts = (uint32_t)rt->sm_count * BLOCKS;
    CUtensorMap map_k{}, map_v{};
    auto go = [&](auto kernel) -> Result {
        TESSL_TRY(smem_opt_in(rt, (const void *)kernel, C::SMEM, what, true));
        return launch_pdl(rt, what, kernel, dim3(sp.p.parts), dim3(C::THREADS), C::SMEM, map_k, map_v, sp);
    };
    if (p.cache.num_pages == 0 || sp.box < 8) return go(attn::attn_paged_split_kernel<DP, false, BLOCKS>);
    TESSL_TRY(cache_maps(rt, what, p.cache, sp.box, &map_k, &map_v));
    return go(attn::attn_paged_split_kernel<DP, true, BLOCKS>);
}

template <int DP>
Result launch_tiles(TesslRuntime *rt, const Params &p, bool negate)
{
    using C = attn::TileCfg<DP>;
    const char *what = "attn_paged tile launch";
    auto kernel = attn::attn_paged_tile_kernel<DP>;
    TESSL_TRY(smem_opt_in(rt, (const void *)kernel, C::SMEM, what, true));
    attn::TileParams tp{p, box_of(p.cache.page_size, attn::kTileKeys), negate};
    tp.p.parts = (uint32_t)rt->sm_count;
    CUtensorMap map_k, map_v;
    TESSL_TRY(cache_maps(rt, what, p.cache, tp.box, &map_k, &map_v));
    return launch_pdl(rt, what, kernel, dim3(tp.p.parts), dim3(C::THREADS), C::SMEM, map_k, map_v, tp);
}

/// A number of 48 bits that no other call's items are counted with: the n-th of a sequence that differs from runtime to runtime (splitmix64).
uint64_t next_mark(TesslRuntime *rt)
{
    if (!rt->attn_mark) {
        std::random_device random;
        rt->attn_mark = ((uint64_t)random() << 32 | random()) ^ (uint64_t)(uintptr_t)rt;
    }
    uint64_t z = rt->attn_mark += 0x9e3779b97f4a7c15ull;
    z = (z ^ (z >> 30)) * 0xbf58476d1ce4e5b9ull;
    z = (z ^ (z >> 27)) * 0x94d049bb133111ebull;
    z = (z ^ (z >> 31)) >> 16;
    return z ? z : 1;  // 0 is nobody's
}

Result heads_validate(const TesslPagedKv &cache, uint32_t total_new, uint32_t n_heads, const char *what)
{
    if (n_heads == 0 || n_heads % cache.n_kv_heads != 0)
        return fmt("%s: n_heads %u is not a multiple of n_kv_heads %u", what, n_heads, cache.n_kv_heads);
    TESSL_TRY(require_i32_extent(elems(total_new, n_heads), "attn_paged: total_new * n_heads"));
    if (elems(n_heads, cache.head_dim) > 0xffffffffull) return fmt("%s: rows of %u heads are too long", what, n_heads);
    return ok();
}

Result attn_params(const TesslPagedKv &cache, const TesslPagedSeqs &seqs, uint32_t total_new, uint32_t n_heads, const char *what, Params *p)
{
    TESSL_TRY(paged::cache_validate(cache, what, &p->cache));
    TESSL_TRY(paged::seqs_validate(seqs, cache, total_new, what, &p->seqs));
    TESSL_TRY(heads_validate(cache, total_new, n_heads, what));
    p->n_heads = n_heads, p->group = attn::Divisor::of(n_heads / cache.n_kv_heads), p->page = attn::Divisor::of(cache.page_size);
    return ok();
}

}  // namespace

namespace nn {

uint64_t attn_paged_workspace_bytes(TesslRuntime *rt, uint32_t total_new, uint32_t n_heads, const TesslPagedKv &cache, const TesslPagedSeqs &seqs)
{
    const char *what = "attn_paged_workspace_bytes";
    if (!paged::cache_sizes_validate(cache, what).empty() || !paged::seqs_sizes_validate(seqs, total_new, what).empty() ||
        !heads_validate(cache, total_new, n_heads, what).empty())
        return 0;
    const uint32_t group = n_heads / cache.n_kv_heads;
    if (too_much(cache, seqs, total_new, group, wants_tiles(cache, seqs, total_new, group))) return 0;
    return workspace_of(rt, cache, seqs, may_want_tiles(cache, seqs, total_new, group));
}

Result attn_paged(TesslRuntime *rt, const TesslBuf &q, const TesslPagedKv &cache, const TesslPagedSeqs &seqs, const TesslBuf &out,
                  const TesslBuf &workspace, uint32_t total_new, uint32_t n_heads, uint32_t q_stride, float scale, bool causal, uint32_t window)
{
    const char *what = "attn_paged";
    Params p{};
    TESSL_TRY(attn_params(cache, seqs, total_new, n_heads, what, &p));
    if (!std::isfinite(scale * 1.4426950408889634f)) return fmt("%s: scale is not finite, or too large", what);
    if (window && !causal) return fmt("%s: a window needs causal attention", what);
    const uint64_t width = elems(n_heads, cache.head_dim);
    uint32_t out_stride = 0;
    TESSL_TRY(paged::rows_validate(q, total_new, width, &q_stride, 2, what, "q"));
    TESSL_TRY(paged::rows_validate(out, total_new, width, &out_stride, 2, what, "out"));
    TESSL_TRY(require_aligned16(q, "attn_paged q"));
    TESSL_TRY(require_aligned16(out, "attn_paged out"));
    if (q_stride % 8 != 0) return fmt("%s: rows of q are %u apart, not a multiple of 8", what, q_stride);
    // A scale of zero makes zeros of scores that a mask has set to -inf: the tile kernel masks before it scales.
    p.scale_log2 = scale * 1.4426950408889634f;
    const bool tiles = wants_tiles(cache, seqs, total_new, p.group.d) && p.scale_log2 != 0.0f;
    if (too_much(cache, seqs, total_new, p.group.d, tiles)) return fmt("%s: more rows and keys than one call counts", what);
    const uint64_t need = workspace_of(rt, cache, seqs, tiles);
    if (workspace.nbytes < need) return fmt("%s: the workspace has %llu bytes, the call needs %llu", what, (unsigned long long)workspace.nbytes, (unsigned long long)need);
    TESSL_TRY(require_aligned16(workspace, "attn_paged workspace"));
    if (!workspace.ptr) return fmt("%s: null workspace", what);
    const Named writes[] = {{"out", &out}, {"workspace", &workspace}};
    const Named reads[] = {{"q", &q}, {"cache k", &cache.k}, {"cache v", &cache.v}, {"page_table", &seqs.page_table},
                           {"kv_lens", &seqs.kv_lens}, {"q_starts", &seqs.q_starts}};
    TESSL_TRY(require_disjoint_writes(what, writes, 2, reads, 6));
    if (total_new == 0 || seqs.num_seqs == 0) return ok();
    p.q = static_cast<const uint16_t *>(q.ptr), p.out = static_cast<uint16_t *>(out.ptr), p.work = static_cast<float *>(workspace.ptr);
    p.q_stride = q_stride;
    if (cache.num_pages == 0) p.cache.k = p.cache.v = static_cast<uint16_t *>(q.ptr);  // copies of no bytes still name an address
    p.causal = causal, p.window = window, p.status = rt->status_dev;
    p.mark = next_mark(rt);
    const bool two = split_blocks(rt, cache, seqs) == 2;
    return with_dim(cache.head_dim, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        if (!tiles) return two ? launch_split<DP, 2>(rt, p) : launch_split<DP, 1>(rt, p);
        const bool negate = p.scale_log2 < 0.0f;
        p.scale_log2 = std::fabs(p.scale_log2);
        return launch_tiles<DP>(rt, p, negate);
    });
}

}  // namespace nn
}  // namespace tessl
