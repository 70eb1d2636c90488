// Attention over a paged cache: checks, routes and launches.
#include <cmath>

#include "attn_paged_split.cuh"

namespace tessl {
namespace {

using attn::Params;

uint32_t padded_dim(uint32_t d) { return d <= 64 ? 64 : d <= 128 ? 128 : d <= 192 ? 192 : 256; }

template <int DP>
size_t split_workspace(const TesslRuntime *rt)
{
    return (size_t)rt->sm_count * 2 * attn::Part<attn::kSplitRows, DP>::FLOATS * sizeof(float);
}

size_t workspace_of(const TesslRuntime *rt, uint32_t head_dim)
{
    switch (padded_dim(head_dim)) {
    case 64: return split_workspace<64>(rt);
    case 128: return split_workspace<128>(rt);
    case 192: return split_workspace<192>(rt);
    default: return split_workspace<256>(rt);
    }
}

template <int DP>
Result launch_split(TesslRuntime *rt, Params p)
{
    using C = attn::SplitCfg<DP>;
    const char *what = "attn_paged launch";
    auto kernel = attn::attn_paged_split_kernel<DP>;
    TESSL_TRY(smem_opt_in(rt, (const void *)kernel, C::SMEM, what, true));
    p.parts = (uint32_t)rt->sm_count;
    p.min_units = 2;
    TESSL_TRY(launch_pdl(rt, what, kernel, dim3(p.parts), dim3(C::THREADS), C::SMEM, p));
    return launch_pdl(rt, what, attn::attn_paged_combine_kernel<attn::kSplitRows, attn::kSplitUnit, DP, 4>, dim3(p.parts - 1, attn::kSplitRows / 4),
                      dim3(128), 0, p);
}

Result attn_params(const TesslPagedKv &cache, const TesslPagedSeqs &seqs, uint32_t total_new, uint32_t n_heads, const char *what, Params *p)
{
    TESSL_TRY(paged::cache_validate(cache, what, &p->cache));
    TESSL_TRY(paged::seqs_validate(seqs, cache, total_new, what, &p->seqs));
    if (n_heads == 0 || n_heads % cache.n_kv_heads != 0)
        return fmt("%s: n_heads %u is not a multiple of n_kv_heads %u", what, n_heads, cache.n_kv_heads);
    TESSL_TRY(require_i32_extent(elems(total_new, n_heads), "attn_paged: total_new * n_heads"));
    p->n_heads = n_heads, p->group = n_heads / cache.n_kv_heads;
    return ok();
}

}  // namespace

namespace nn {

uint64_t attn_paged_workspace_bytes(TesslRuntime *rt, uint32_t total_new, uint32_t n_heads, const TesslPagedKv &cache, const TesslPagedSeqs &seqs)
{
    (void)seqs;
    if (cache.head_dim == 0 || cache.head_dim % 8 != 0 || cache.head_dim > 256 || cache.n_kv_heads == 0 || n_heads == 0 ||
        n_heads % cache.n_kv_heads != 0 || elems(total_new, n_heads) > 0x7fffffffull)
        return 0;
    return workspace_of(rt, cache.head_dim);
}

Result attn_paged(TesslRuntime *rt, const TesslBuf &q, const TesslPagedKv &cache, const TesslPagedSeqs &seqs, const TesslBuf &out,
                  const TesslBuf &workspace, uint32_t total_new, uint32_t n_heads, uint32_t q_stride, float scale, bool causal, uint32_t window)
{
    const char *what = "attn_paged";
    Params p{};
    TESSL_TRY(attn_params(cache, seqs, total_new, n_heads, what, &p));
    if (!std::isfinite(scale)) return fmt("%s: scale is not finite", what);
    if (window && !causal) return fmt("%s: a window needs causal attention", what);
    const uint64_t width = elems(n_heads, cache.head_dim);
    uint32_t out_stride = 0;
    TESSL_TRY(paged::rows_validate(q, total_new, width, &q_stride, 2, what, "q"));
    TESSL_TRY(paged::rows_validate(out, total_new, width, &out_stride, 2, what, "out"));
    TESSL_TRY(require_aligned16(q, "attn_paged q"));
    TESSL_TRY(require_aligned16(out, "attn_paged out"));
    if (q_stride % 8 != 0) return fmt("%s: rows of q are %u apart, not a multiple of 8", what, q_stride);
    const uint64_t need = workspace_of(rt, cache.head_dim);
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
    p.scale_log2 = scale * 1.4426950408889634f;
    p.causal = causal, p.window = window, p.status = rt->status_dev;
    switch (padded_dim(cache.head_dim)) {
    case 64: return launch_split<64>(rt, p);
    case 128: return launch_split<128>(rt, p);
    case 192: return launch_split<192>(rt, p);
    default: return launch_split<256>(rt, p);
    }
}

}  // namespace nn
}  // namespace tessl
