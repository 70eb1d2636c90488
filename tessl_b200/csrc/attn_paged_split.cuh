// Attention of few rows per key head (single tokens, short chunks) over a paged cache.
//
// One pass over the keys with the running maximum and sum of the softmax. An item is 16 rows (the M of mma.sync m16n8k16) of
// one sequence and key head; a part of its keys belongs to a block (attn_paged_common.cuh), whose warps take steps of 16 keys
// in turn. A warp has its own ring of steps in shared memory, filled with cp.async 16 bytes at a time (rows of K and V at
// swizzled chunks, keys that do not exist as zeros), its own maxima, sums and 16 x D accumulators in registers, so nothing but
// its own copies makes it wait; the warps meet at the end of the item's part.
//
// The weights p of a step are rounded to bf16 for the product with V: relative 2^-9 each, independent, against the 2^-9 of the
// output's own rounding; their sum is taken in f32 before that.
//
// Bound by memory: a step of 16 keys is 64 D bytes and D / 2 MMAs of 16 x 8 x 16.
#pragma once
#include "attn_paged_common.cuh"

namespace tessl {
namespace attn {

constexpr uint32_t kSplitRows = 16, kSplitUnit = 64, kStep = 16;

template <int DP>
struct SplitCfg {
    static constexpr uint32_t WARPS = DP <= 128 ? 8 : 4, THREADS = WARPS * 32;
    static constexpr uint32_t ROW = DP * 2, TILE = kStep * ROW, STAGE = 2 * TILE;  // bytes
    static constexpr uint32_t STAGES = DP == 64 ? 6 : DP == 192 ? 4 : 3;
    static constexpr uint32_t RING = STAGES * STAGE;
    static constexpr uint32_t Q_BYTES = kSplitRows * ROW;
    static constexpr uint32_t MASK_BYTES = WARPS * STAGES * 4, ML_BYTES = WARPS * kSplitRows * 8;
    static constexpr uint32_t SMEM = WARPS * RING + Q_BYTES + MASK_BYTES + ML_BYTES;
    static_assert(RING >= kSplitRows * DP * 4, "a warp's accumulators lie in its ring when warps meet");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t a, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
/// Byte offset of 16-byte chunk c of row r in a tile with rows of DP bf16: chunks of eight rows fall on different banks.
template <int DP>
__device__ __forceinline__ uint32_t chunk_at(uint32_t r, uint32_t c)
{
    return r * (DP * 2) + ((c ^ (r & 7u)) << 4);
}

template <int DP>
__global__ void __launch_bounds__(SplitCfg<DP>::THREADS, 1) attn_paged_split_kernel(const Params p)
{
    using C = SplitCfg<DP>;
    constexpr uint32_t ROWS = kSplitRows, UNIT = kSplitUnit;
    asm volatile("griddepcontrol.launch_dependents;");
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t ring = q4k::smem_u32(smem) + warp * C::RING;
    const uint32_t q_smem = q4k::smem_u32(smem) + C::WARPS * C::RING;
    uint32_t *masks = reinterpret_cast<uint32_t *>(smem + C::WARPS * C::RING + C::Q_BYTES) + warp * C::STAGES;
    float2 *ml = reinterpret_cast<float2 *>(smem + C::WARPS * C::RING + C::Q_BYTES + C::MASK_BYTES);  // [warp][row]
    const uint32_t d = p.cache.head_dim, chunks = d / 8;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    using L = Line<ROWS, UNIT, C::THREADS>;
    __shared__ typename L::Shared shared;
    L line;
    Cursor cur;
    uint64_t u;
    if (!line.start(p, blockIdx.x, shared, u, cur)) return;
    const uint64_t u_end = line.cut(blockIdx.x + 1);
    if (u >= u_end) return;

    while (true) {
        const uint32_t n_units = (uint32_t)min((uint64_t)(cur.units - cur.u0), u_end - u);
        const Seq &seq = cur.seq;
        const uint32_t kv_head = cur.kv_head, u0 = cur.u0, rows = seq.news * p.group, row0 = cur.block * ROWS;
        // Keys of this part that the block's rows may see.
        const uint32_t i0 = row0 / p.group, i1 = (min(row0 + ROWS, rows) - 1) / p.group;
        uint32_t lo, hi;
        key_range(p, seq, i0, i1, lo, hi);
        const uint32_t key0 = max((cur.first + u0) * UNIT, lo / kStep * kStep), key1 = min((cur.first + u0 + n_units) * UNIT, hi);
        const uint32_t steps = key1 > key0 ? (key1 - key0 + kStep - 1) / kStep : 0;
        const uint32_t mine = steps > warp ? (steps - warp + C::WARPS - 1) / C::WARPS : 0;

        // Q rows, zeros past the last row and column.
        for (uint32_t c = tid; c < ROWS * (DP / 8); c += C::THREADS) {
            const uint32_t r = c / (DP / 8), cc = c % (DP / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row0 + r < rows && cc < chunks) {
                uint32_t token, head;
                row_at(p, seq, kv_head, row0 + r, token, head);
                v = __ldcg(reinterpret_cast<const uint4 *>(p.q + (size_t)token * p.q_stride + (size_t)head * d + cc * 8));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(q_smem + chunk_at<DP>(r, cc)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }

        const int32_t *table = p.seqs.table + (size_t)seq.index * p.seqs.max_pages;
        const size_t head_off = (size_t)kv_head * p.cache.head_stride;
        // Lane l of a warp knows where key l % 16 of a step lies: -1 where there is none.
        auto locate = [&](uint32_t j) -> int64_t {
            const uint32_t key = key0 + (warp + j * C::WARPS) * kStep + (lane & 15u);
            if (j >= mine || key >= key1) return -1;
            const uint32_t page = (uint32_t)__ldcg(table + key / p.cache.page_size);
            if (page >= p.cache.num_pages) return -1;
            return (int64_t)(page * p.cache.page_stride + (uint64_t)(key % p.cache.page_size) * p.cache.token_stride + head_off);
        };
        auto request = [&](uint32_t j, int64_t at) {  // step j of this warp into stage j % STAGES
            const uint32_t stage = j % C::STAGES, dst = ring + stage * C::STAGE;
            const uint32_t live = __ballot_sync(0xffffffffu, at >= 0) & 0xffffu;
            if (lane == 0) masks[stage] = live;
#pragma unroll 4
            for (uint32_t c = lane; c < kStep * (DP / 8); c += 32) {
                const uint32_t r = c / (DP / 8), cc = c % (DP / 8);
                const int64_t row = __shfl_sync(0xffffffffu, at, r);
                const bool ok = row >= 0 && cc < chunks;
                const size_t off = ok ? (size_t)row + cc * 8 : 0;
                cp_async16(dst + chunk_at<DP>(r, cc), p.cache.k + off, ok);
                cp_async16(dst + C::TILE + chunk_at<DP>(r, cc), p.cache.v + off, ok);
            }
        };
#pragma unroll
        for (uint32_t j = 0; j < C::STAGES - 1; ++j) {
            if (j < mine) request(j, locate(j));
            cp_async_commit();
        }
        int64_t next = locate(C::STAGES - 1);
        __syncthreads();  // Q is there

        constexpr bool Q_REGS = DP <= 128;
        uint32_t qf[Q_REGS ? DP / 16 : 1][4];
        // A of k-slice k: rows lane % 16, columns 16 k + 8 (lane / 16)
        auto q_frag = [&](uint32_t k, uint32_t (&f)[4]) { ldsm4(q_smem + chunk_at<DP>(lane & 15u, 2 * k + (lane >> 4)), f); };
        if constexpr (Q_REGS) {
#pragma unroll
            for (uint32_t k = 0; k < DP / 16; ++k) q_frag(k, qf[k]);
        }
        float o[DP / 8][4];
#pragma unroll
        for (uint32_t n = 0; n < DP / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        // This lane's two rows: lane / 4 and 8 more.
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        uint32_t lo_r[2], hi_r[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t r = row0 + lane / 4 + 8 * h;
            const uint32_t i = min(r, rows - 1) / p.group;
            key_range(p, seq, i, i, lo_r[h], hi_r[h]);
        }
        uint32_t lo_all, hi_all;  // what every row of the block sees
        {
            uint32_t t;
            key_range(p, seq, i1, i1, lo_all, t);
            key_range(p, seq, i0, i0, t, hi_all);
        }

        for (uint32_t j = 0; j < mine; ++j) {
            cp_async_wait<C::STAGES - 2>();
            __syncwarp();
            const uint32_t stage = j % C::STAGES, kt = ring + stage * C::STAGE, vt = kt + C::TILE;
            const uint32_t key = key0 + (warp + j * C::WARPS) * kStep, live = masks[stage];
            if (j + C::STAGES - 1 < mine) request(j + C::STAGES - 1, next);
            cp_async_commit();
            next = locate(j + C::STAGES);

            float sc[2][4] = {};
#pragma unroll
            for (uint32_t k = 0; k < DP / 16; ++k) {
                uint32_t a[4], b[4];
                if constexpr (Q_REGS) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) a[x] = qf[k][x];
                } else {
                    q_frag(k, a);
                }
                // keys 0-7 then 8-15, columns 16 k and 8 more
                ldsm4(kt + chunk_at<DP>((lane & 7u) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1u)), b);
                mma_bf16(sc[0], a, b[0], b[1]);
                mma_bf16(sc[1], a, b[2], b[3]);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[n][x] *= p.scale_log2;
            if (live != 0xffffu || key < lo_all || key + kStep > hi_all) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t t = 8 * n + 2 * (lane & 3u) + (x & 1);
                        if (!((live >> t) & 1u) || key + t < lo_r[x >> 1] || key + t >= hi_r[x >> 1]) sc[n][x] = -INFINITY;
                    }
            }
            float scale_o[2];
            bool grew = false;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float t = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                t = fmaxf(t, m[h]);
                const float top = t == -INFINITY ? 0.0f : t;
                scale_o[h] = exp2_fast(m[h] - top);
                grew |= t != m[h];
                m[h] = t;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) sc[n][2 * h + x] = exp2_fast(sc[n][2 * h + x] - top), sum += sc[n][2 * h + x];
                l[h] = l[h] * scale_o[h] + sum;
            }
            if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                for (uint32_t n = 0; n < DP / 8; ++n) o[n][0] *= scale_o[0], o[n][1] *= scale_o[0], o[n][2] *= scale_o[1], o[n][3] *= scale_o[1];
            }
            const uint32_t pf[4] = {bf16_pair(sc[0][0], sc[0][1]), bf16_pair(sc[0][2], sc[0][3]), bf16_pair(sc[1][0], sc[1][1]), bf16_pair(sc[1][2], sc[1][3])};
#pragma unroll
            for (uint32_t n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                // keys 0-7, 8-15 of columns 16 n, then of 8 more
                ldsm4_t(vt + chunk_at<DP>(lane & 15u, 2 * n + (lane >> 4)), b);
                mma_bf16(o[2 * n], pf, b[0], b[1]);
                mma_bf16(o[2 * n + 1], pf, b[2], b[3]);
            }
            __syncwarp();  // the stage is read
        }
        cp_async_wait<0>();

        // ---- the warps meet: sums to the block's maximum, every warp's accumulators in its ring ----
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3u) == 0) ml[warp * ROWS + lane / 4 + 8 * h] = make_float2(m[h], l[h]);
        }
        __syncthreads();
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float t = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < C::WARPS; ++w) t = fmaxf(t, ml[w * ROWS + lane / 4 + 8 * h].x);
            top[h] = t;
            const float f = m[h] == -INFINITY ? 0.0f : exp2_fast(m[h] - t);
            float *dst = reinterpret_cast<float *>(smem + warp * C::RING) + (lane / 4 + 8 * h) * DP;
#pragma unroll
            for (uint32_t n = 0; n < DP / 8; ++n)  // 16-byte chunks swizzled: eight rows on different banks
                *reinterpret_cast<float2 *>(dst + (((2 * n + ((lane >> 1) & 1u)) ^ (lane / 4)) << 2) + (lane & 1u) * 2) =
                    make_float2(o[n][2 * h] * f, o[n][2 * h + 1] * f);
        }
        __syncthreads();
        const bool whole = n_units == cur.units;
        using P = Part<ROWS, DP>;
        float *part = P::at(p.work, blockIdx.x, u0 == 0);
        for (uint32_t c = tid; c < ROWS * (DP / 4); c += C::THREADS) {
            const uint32_t r = c / (DP / 4), x = c % (DP / 4);
            if (row0 + r >= rows || x * 4 >= d) continue;
            float4 sum = make_float4(0, 0, 0, 0);
            float t = -INFINITY, den = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < C::WARPS; ++w) {
                const float4 v = *reinterpret_cast<const float4 *>(smem + w * C::RING + (size_t)r * DP * 4 + ((x ^ (r & 7u)) << 4));
                sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                t = fmaxf(t, ml[w * ROWS + r].x);
            }
#pragma unroll
            for (uint32_t w = 0; w < C::WARPS; ++w) {
                const float2 v = ml[w * ROWS + r];
                if (v.x != -INFINITY) den += v.y * exp2_fast(v.x - t);
            }
            if (whole) {
                const float inv = den == 0.0f ? 0.0f : 1.0f / den;
                uint32_t token, head;
                row_at(p, seq, kv_head, row0 + r, token, head);
                *reinterpret_cast<uint2 *>(p.out + ((size_t)token * p.n_heads + head) * d + x * 4) =
                    make_uint2(bf16_pair(sum.x * inv, sum.y * inv), bf16_pair(sum.z * inv, sum.w * inv));
            } else {
                *reinterpret_cast<float4 *>(part + P::four(r, x)) = sum;
                if (x == 0) part[P::TOP + r] = t, part[P::SUM + r] = den;
            }
        }
        u += n_units;
        if (u >= u_end) return;
        L::next(p, cur);
        __syncthreads();  // rings, Q and ml are read
    }
}

}  // namespace attn
}  // namespace tessl
