// What the attention kernels over a paged cache share: the launch parameters, the ranges of keys that rows see, and the division
// of a call's work among the blocks of a launch.
//
// The rows of one sequence and key head are its new tokens times the `group` query heads that read that key head, token by
// token: they all multiply the same keys. A block of rows of them is an item, its keys come in units, and all units of the
// call, item after item, are one line that is cut into equal parts, one per block of the launch: whatever the lengths of the
// sequences, every block reads the same number of keys. The lengths are on the device, so the blocks work the cuts out
// themselves. A block that has an item to itself writes its rows; the parts of an item that a cut divides go to the workspace,
// two at most per block (the end of one item, the start of another), and a second launch, one block per cut, adds them up in the
// order of the keys: the same sums on every run.
#pragma once
#include "paged_common.cuh"
#include "q4_gemv_tma.cuh"

namespace tessl {
namespace attn {

struct Params {
    const uint16_t *q;
    uint16_t *out;
    float *work;
    paged::Cache cache;
    paged::Seqs seqs;
    uint32_t q_stride, n_heads, group;
    float scale_log2;  // scale * log2 e
    uint32_t causal, window;
    uint32_t parts;      // blocks that the line of units may be cut for
    uint32_t min_units;  // units that a part is worth
    uint32_t *status;
};

/// One sequence as its rows see it.
struct Seq {
    uint32_t index, row0, news;  // its new tokens are rows row0 .. row0 + news - 1 of the call
    uint32_t keys;               // tokens that have a slot
    int32_t base;                // position of its first new token
};

__device__ __forceinline__ Seq seq_at(const Params &p, uint32_t s)
{
    Seq q;
    q.index = s;
    q.row0 = paged::start_of(p.seqs, s);
    const uint32_t end = paged::start_of(p.seqs, s + 1);
    q.news = end > q.row0 ? end - q.row0 : 0;
    const uint32_t len = paged::len_of(p.seqs, s);
    q.keys = (uint32_t)min((uint64_t)len, p.seqs.capacity);
    q.base = (int32_t)(len - q.news);
    return q;
}

/// Keys [lo, hi) outside of which tokens i0 .. i1 of a sequence see nothing.
__device__ __forceinline__ void key_range(const Params &p, const Seq &q, uint32_t i0, uint32_t i1, uint32_t &lo, uint32_t &hi)
{
    lo = 0, hi = q.keys;
    if (p.causal) {
        hi = (uint32_t)min(max((int64_t)q.base + i1 + 1, (int64_t)0), (int64_t)q.keys);
        if (p.window) lo = (uint32_t)min(max((int64_t)q.base + i0 + 1 - p.window, (int64_t)0), (int64_t)hi);
    }
}

/// How a sequence divides: blocks of ROWS rows, units of UNIT keys from `first` on for each of them.
struct Extent {
    uint32_t blocks, units, first;
};
template <uint32_t ROWS, uint32_t UNIT>
__device__ __forceinline__ Extent extent_of(const Params &p, const Seq &q)
{
    Extent e{0, 0, 0};
    if (q.news == 0) return e;
    uint32_t lo, hi;
    key_range(p, q, 0, q.news - 1, lo, hi);
    e.blocks = (uint32_t)(((uint64_t)q.news * p.group + ROWS - 1) / ROWS);
    e.first = lo / UNIT * UNIT;
    e.units = max(1u, (hi - e.first + UNIT - 1) / UNIT);  // rows that see nothing are written too
    return e;
}
template <uint32_t ROWS, uint32_t UNIT>
__device__ __forceinline__ uint64_t cost_of(const Params &p, uint32_t s)
{
    const Extent e = extent_of<ROWS, UNIT>(p, seq_at(p, s));
    return (uint64_t)e.blocks * e.units * p.cache.n_kv_heads;
}

/// The line of units and how it is cut.
struct Line {
    uint64_t total;
    uint32_t parts;
    __device__ __forceinline__ uint64_t cut(uint32_t c) const { return total / parts * c + total % parts * c / parts; }
    /// The part that holds unit u.
    __device__ __forceinline__ uint32_t part_of(uint64_t u) const
    {
        uint32_t c = (uint32_t)min((uint64_t)parts - 1, (uint64_t)((double)u / (double)total * parts));
        while (c > 0 && cut(c) > u) --c;
        while (c + 1 < parts && cut(c + 1) <= u) ++c;
        return c;
    }
};

/// Sum of v over the threads in front of this one, and over the block's in `total`.
template <uint32_t THREADS>
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t *scratch, uint64_t &total)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t s = v;
#pragma unroll
    for (uint32_t o = 1; o < 32; o *= 2) {
        const uint64_t t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();  // scratch may still be read
    if (lane == 31) scratch[warp] = s;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += scratch[w];
        total += scratch[w];
    }
    return before + s - v;
}

template <uint32_t ROWS, uint32_t UNIT, uint32_t THREADS>
__device__ __forceinline__ Line line_of(const Params &p, uint64_t *scratch)
{
    uint64_t sum = 0;
    for (uint32_t s = threadIdx.x; s < p.seqs.num_seqs; s += THREADS) sum += cost_of<ROWS, UNIT>(p, s);
    Line l;
    block_scan<THREADS>(sum, scratch, l.total);
    l.parts = (uint32_t)min((uint64_t)p.parts, max((uint64_t)1, l.total / p.min_units));
    return l;
}

/// The sequence that holds unit u of the line, and the unit at which it starts. The whole block calls this.
template <uint32_t ROWS, uint32_t UNIT, uint32_t THREADS>
__device__ __forceinline__ uint32_t seq_of_unit(const Params &p, uint64_t u, uint64_t *scratch, uint64_t &start)
{
    __shared__ uint32_t found;
    __shared__ uint64_t found_start;
    uint64_t before = 0;
    if (threadIdx.x == 0) found = p.seqs.num_seqs;
    for (uint32_t s0 = 0; s0 < p.seqs.num_seqs; s0 += THREADS) {
        const uint32_t s = s0 + threadIdx.x;
        const uint64_t cost = s < p.seqs.num_seqs ? cost_of<ROWS, UNIT>(p, s) : 0;
        uint64_t total;
        const uint64_t at = before + block_scan<THREADS>(cost, scratch, total);
        if (at <= u && u < at + cost) found = s, found_start = at;
        before += total;
        __syncthreads();
        if (u < before) break;
    }
    __syncthreads();
    start = found_start;
    const uint32_t s = found;
    __syncthreads();
    return s;
}

/// A part of an item in the workspace: 16 rows of DP unnormalised sums, then the rows' maxima (in powers of two) and sums.
template <uint32_t ROWS, uint32_t DP>
struct Part {
    static constexpr uint32_t FLOATS = ROWS * DP + 2 * ROWS;
    /// `head`: the start of an item, else its middle or end.
    static __device__ __forceinline__ float *at(float *work, uint32_t part, bool head) { return work + ((size_t)part * 2 + head) * FLOATS; }
};

__device__ __forceinline__ float exp2_fast(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

/// Row r of a sequence and key head: its row of q and out, in heads.
__device__ __forceinline__ void row_at(const Params &p, const Seq &q, uint32_t kv_head, uint32_t r, uint32_t &token, uint32_t &head)
{
    token = r / p.group;
    head = kv_head * p.group + (r - token * p.group);
    token += q.row0;
}

/// Adds up the parts of the items that cuts divide, one block per cut and ROWS_PER rows: the first cut in an item does it.
template <uint32_t ROWS, uint32_t UNIT, uint32_t DP, uint32_t ROWS_PER>
__global__ void __launch_bounds__(128) attn_paged_combine_kernel(const Params p)
{
    constexpr uint32_t THREADS = 128;
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ uint64_t scratch[THREADS / 32];
    const Line l = line_of<ROWS, UNIT, THREADS>(p, scratch);
    const uint32_t c = blockIdx.x + 1;
    if (c >= l.parts) return;
    const uint64_t u = l.cut(c);
    uint64_t start;
    const uint32_t s = seq_of_unit<ROWS, UNIT, THREADS>(p, u, scratch, start);
    if (s >= p.seqs.num_seqs) return;
    const Seq q = seq_at(p, s);
    const Extent e = extent_of<ROWS, UNIT>(p, q);
    const uint32_t item = (uint32_t)((u - start) / e.units);
    const uint64_t from = start + (uint64_t)item * e.units, to = from + e.units;
    if (u == from || l.cut(c - 1) > from) return;  // between two items; or an earlier cut is in this one
    const uint32_t kv_head = item / e.blocks, block = item % e.blocks;
    const uint32_t last = l.part_of(to - 1), rows = q.news * p.group, d = p.cache.head_dim;
    constexpr uint32_t LANES = THREADS / ROWS_PER;  // per row
    const uint32_t r = blockIdx.y * ROWS_PER + threadIdx.x / LANES, row = block * ROWS + r;
    if (row >= rows) return;
    float m = -INFINITY;
    for (uint32_t k = c - 1; k <= last; ++k) m = fmaxf(m, __ldcg(Part<ROWS, DP>::at(p.work, k, k == c - 1) + ROWS * DP + r));
    const float top = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    for (uint32_t k = c - 1; k <= last; ++k) {
        const float *a = Part<ROWS, DP>::at(p.work, k, k == c - 1) + ROWS * DP + r;
        sum += __ldcg(a + ROWS) * exp2_fast(__ldcg(a) - top);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint32_t token, head;
    row_at(p, q, kv_head, row, token, head);
    uint16_t *out = p.out + ((size_t)token * p.n_heads + head) * d;
    for (uint32_t x = (threadIdx.x % LANES) * 4; x < d; x += LANES * 4) {
        float4 o = make_float4(0, 0, 0, 0);
        for (uint32_t k = c - 1; k <= last; ++k) {
            const float *a = Part<ROWS, DP>::at(p.work, k, k == c - 1);
            const float f = exp2_fast(__ldcg(a + ROWS * DP + r) - top);
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(a + r * DP + x));
            o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
        }
        *reinterpret_cast<uint2 *>(out + x) = make_uint2(bf16_pair(o.x * inv, o.y * inv), bf16_pair(o.z * inv, o.w * inv));
    }
}

}  // namespace attn
}  // namespace tessl
