// Attention of few rows per key head (single tokens, short chunks) over a paged cache.
//
// One pass over the keys with the running maximum and sum of the softmax. An item is 16 rows (the M of mma.sync m16n8k16) of
// one sequence and key head; a part of its keys belongs to a block (attn_paged_common.cuh), whose warps take steps of 16 keys
// in turn. A warp has its own ring of tiles (16 keys of K, of V) in shared memory, its own maxima, sums and 16 x D accumulators in
// registers, so nothing but its own copies makes it wait; the warps meet at the end of the item's part.
//
// Tiles come by TMA, 64 columns wide with the 128-byte swizzle, which is also what ldmatrix reads without bank conflicts: a tile
// is one or two copies per 64 columns where pages are a multiple of eight tokens. Other pages, by row, with cp.async. (Rows with
// cp.async throughout: 32 address computations and copies per lane and step of 16 x 128, 4.7 TB/s over 130001 keys and 3.8 TB/s
// of wide heads, where the instructions of four warps bounded it.)
//
// The weights p of a step are rounded to bf16 for the product with V: relative 2^-8 at most, each its own way, against the 2^-8 of
// the output's own rounding; their sum is taken in f32 before that.
//
// Bound by memory: a step of 16 keys is 64 D bytes and D / 4 MMAs of 16 x 8 x 16. 32 heads of 128 on 8, a token over 130001 keys: 102 us,
// 5.2 TB/s; 64 tokens over up to 12000 keys each: 287 us, 5.6 TB/s, of 6.6 that a copy reaches (call behind call 273 us). Over a few hundred keys the time is
// latency: 2 us to the first request (lengths, then page ids), 1 us to the first tile, 0.7 us for the warps to meet, 4 us to join parts.
#pragma once
#include "attn_paged_common.cuh"

namespace tessl {
namespace attn {

constexpr uint32_t kSplitRows = 16, kSplitUnit = 64, kStep = 16;
// What a second part of an item costs, in units: a token over 400 keys (7 units) took 9.3 us whole and 10.9 us cut, over 777 keys (13 units)
// 13.7 us and 11.6 us.
constexpr uint32_t kSplitExtra = 9;

/// BLOCKS: of an SM at a time.
template <int DP, int BLOCKS>
struct SplitCfg {
    static constexpr uint32_t WARPS = 8 / BLOCKS, THREADS = WARPS * 32;
    static constexpr uint32_t CHUNKS = DP / 64;            // 64-column chunks of a row
    static constexpr uint32_t CHUNK = kStep * 128, TILE = CHUNKS * CHUNK;  // bytes
    static constexpr uint32_t SLOTS = 24576 / TILE;        // of a warp's ring: 12, 6, 4, 3
    static constexpr uint32_t RING = SLOTS * TILE;
    static constexpr uint32_t Q_BYTES = kSplitRows * DP * 2;
    static constexpr uint32_t ML_BYTES = WARPS * kSplitRows * 8, BAR_BYTES = WARPS * SLOTS * 8;
    static constexpr uint32_t SMEM = WARPS * RING + Q_BYTES + ML_BYTES + BAR_BYTES;
    static_assert(RING >= kSplitRows * DP * 4, "a warp's accumulators lie in its ring when warps meet");
};

struct SplitParams {
    Params p;
    uint32_t box;  // tokens per TMA box: 8 or 16
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
/// Box of the cache: 64 columns of one key head, some tokens of one page.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
        "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
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
/// Byte offset of 16-byte piece c of row r of a tile of 16 rows: 64-column chunks one behind the other, 128-byte swizzle.
__device__ __forceinline__ uint32_t piece_at(uint32_t r, uint32_t c) { return (c >> 3) * (kStep * 128) + r * 128 + (((c ^ r) & 7u) << 4); }

template <int DP, bool TMA, int BLOCKS>
__global__ void __launch_bounds__(SplitCfg<DP, BLOCKS>::THREADS, BLOCKS)
    attn_paged_split_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SplitParams sp)
{
    using C = SplitCfg<DP, BLOCKS>;
    using P = Part<kSplitRows, DP>;
    constexpr uint32_t ROWS = kSplitRows, UNIT = kSplitUnit, SLOTS = C::SLOTS;
    asm volatile("griddepcontrol.launch_dependents;");
    const Params &p = sp.p;
    extern __shared__ __align__(1024) uint8_t smem[];
    using L = Line<ROWS, UNIT, C::THREADS, kSplitExtra>;
    __shared__ typename L::Shared shared;
    __shared__ Pending pending[2];
    __shared__ int abort_flag, made_finite;
    __shared__ uint32_t came[2];
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t ring = q4k::smem_u32(smem) + warp * C::RING, q_smem = q4k::smem_u32(smem) + C::WARPS * C::RING;
    float2 *ml = reinterpret_cast<float2 *>(smem + C::WARPS * C::RING + C::Q_BYTES);  // [warp][row]
    const uint32_t bars = q_smem + C::Q_BYTES + C::ML_BYTES + warp * SLOTS * 8;
    const uint32_t d = p.cache.head_dim, pieces = d / 8;
    volatile int *abortp = &abort_flag;
    if (tid == 0) abort_flag = 0, made_finite = 0;
    if (TMA && lane == 0) {
        for (uint32_t s = 0; s < SLOTS; ++s) q4k::mbar_init(bars + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        if (warp == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
        }
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (TMA) asm volatile("fence.proxy.async.global;" ::: "memory");  // ordinary stores of the launch in front, read by the copy engine

    L line;
    Cursor cur;
    uint32_t u;
    if (!line.start(p, blockIdx.x, shared, u, cur)) return;
    const uint32_t u_end = line.cut(blockIdx.x + 1);
    if (u >= u_end) return;
    bool has[2] = {false, false};
    uint32_t at = 0, phases = 0;  // the ring's next slot, the parity of each slot's next phase

    while (true) {
        const uint32_t n_units = line.units_to(cur, u, u_end);
        const Seq &seq = cur.seq;
        const uint32_t kv_head = cur.kv_head, u0 = cur.u0, rows = seq.news * p.group.d, row0 = cur.block * ROWS;
        // Keys of this part that the block's rows may see.
        const uint32_t i0 = p.group.div(row0), i1 = p.group.div(min(row0 + ROWS, rows) - 1);
        uint32_t lo, hi;
        key_range(p, seq, i0, i1, lo, hi);
        const uint32_t key0 = max((cur.first + u0) * UNIT, lo / kStep * kStep), key1 = min((cur.first + u0 + n_units) * UNIT, hi);
        const uint32_t steps = key1 > key0 ? (key1 - key0 + kStep - 1) / kStep : 0;
        const uint32_t mine = steps > warp ? (steps - warp + C::WARPS - 1) / C::WARPS : 0;
        auto key_of = [&](uint32_t j) { return key0 + (warp + j * C::WARPS) * kStep; };

        const int32_t *table = p.seqs.table + (size_t)seq.index * p.seqs.max_pages;
        const uint32_t boxes = TMA ? kStep / sp.box : kStep, span = TMA ? sp.box : 1;
        // Where the tokens of a step lie. TMA: lane l < boxes has the page of box l. Rows: lane l % 16 that of a row, as an offset.
        struct Where {
            uint32_t page, slot;  // page = num_pages: there is none
        };
        auto find = [&](uint32_t j) {
            Where w{p.cache.num_pages, 0};
            const uint32_t l = TMA ? lane : lane & 15u, key = key_of(j) + l * span;
            if (j < mine && l < boxes && key < (TMA ? seq.keys : key1)) {
                const uint32_t page = (uint32_t)__ldcg(table + p.page.div(key));
                if (page < p.cache.num_pages) w.page = page, w.slot = p.page.mod(key);
            }
            return w;
        };
        // The tile of K or V of a step into slot `to`.
        auto request = [&](const Where &w, bool v, uint32_t to) {
            const uint32_t dst = ring + to * C::TILE;
            if constexpr (TMA) {
                if (lane == 0) q4k::mbar_expect_tx(bars + 8 * to, C::TILE);
                __syncwarp();
                if (lane < boxes) {
#pragma unroll
                    for (uint32_t c = 0; c < C::CHUNKS; ++c)
                        tma_load_4d(dst + c * C::CHUNK + lane * sp.box * 128, v ? &map_v : &map_k, (int)(c * 64), (int)kv_head, (int)w.slot, (int)w.page,
                                    bars + 8 * to);
                }
            } else {
                const uint16_t *base = v ? p.cache.v : p.cache.k;
#pragma unroll 4
                for (uint32_t c = lane; c < kStep * (DP / 8); c += 32) {
                    const uint32_t r = c / (DP / 8), cc = c % (DP / 8);
                    const uint32_t page = __shfl_sync(0xffffffffu, w.page, r), slot = __shfl_sync(0xffffffffu, w.slot, r);
                    const bool ok = page < p.cache.num_pages && cc < pieces;
                    const size_t off = page * p.cache.page_stride + (uint64_t)slot * p.cache.token_stride + (uint64_t)kv_head * p.cache.head_stride + cc * 8;
                    cp_async16(dst + piece_at(r, cc), base + (ok ? off : 0), ok);
                }
                cp_async_commit();
            }
        };
        // Tiles K_0, V_0, K_1, ... of this warp go into the ring one behind the other. `holes`: for each of the steps that are on their way,
        // the boxes that are not there, two bits at step % 16 (rows: any row of any step).
        uint32_t holes = 0;
        bool row_hole = false;
        uint32_t issued = 0, done = 0, to = at;  // tiles asked for, tiles that have arrived, the slot of the next one
        Where w = find(0), next = find(1);       // of the step whose tile is asked for next, and of the one behind it
        auto feed = [&](uint32_t most) {
#pragma unroll 2
            for (uint32_t i = 0; i < most; ++i) {
                if (issued < 2 * mine && issued - done < SLOTS) {
                    const uint32_t j = issued / 2;
                    if (issued % 2 == 0) {
                        if constexpr (TMA) {
                            const uint32_t gone = __ballot_sync(0xffffffffu, lane < boxes && w.page >= p.cache.num_pages);
                            holes = (holes & ~(3u << (j % 16 * 2))) | (gone << (j % 16 * 2));
                        } else {
                            row_hole |= __any_sync(0xffffffffu, w.page >= p.cache.num_pages);
                        }
                        request(w, false, to);
                    } else {
                        request(w, true, to);
                        w = next;
                        next = find(j + 2);
                    }
                    ++issued;
                    if (++to == SLOTS) to = 0;
                } else if (!TMA) {
                    cp_async_commit();
                }
            }
        };
        // TMA: the first step only. 45 bytes a clock come out of the copy engine's requests, and a whole ring of every warp in front of the first
        // step held that up by 4000 clocks; the rest is asked for behind it. Rows: a group for every slot (arrived() counts them).
        feed(TMA ? 2 : SLOTS);

        const bool whole = n_units == cur.units;
        if (!whole) {
            has[u0 == 0] = true;
            if (tid == C::THREADS - 32) pending[u0 == 0] = Pending{cur, u - u0}, expect_parts<DP, ROWS>(p, line, u - u0);
        }

        // Q rows, zeros past the last row and column.
        for (uint32_t c = tid; c < ROWS * (DP / 8); c += C::THREADS) {
            const uint32_t r = c / (DP / 8), cc = c % (DP / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (row0 + r < rows && cc < pieces) {
                uint32_t token, head;
                row_at(p, seq, kv_head, row0 + r, token, head);
                v = __ldcg(reinterpret_cast<const uint4 *>(p.q + (size_t)token * p.q_stride + (size_t)head * d + cc * 8));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(q_smem + piece_at(r, cc)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
        }
        __syncthreads();  // Q is there

        constexpr bool Q_REGS = DP <= 128;
        uint32_t qf[Q_REGS ? DP / 16 : 1][4];
        // A of k-slice k: rows lane % 16, columns 16 k + 8 (lane / 16)
        auto q_frag = [&](uint32_t k, uint32_t (&f)[4]) { ldsm4(q_smem + piece_at(lane & 15u, 2 * k + (lane >> 4)), f); };
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
            const uint32_t i = p.group.div(min(row0 + lane / 4 + 8 * h, rows - 1));
            key_range(p, seq, i, i, lo_r[h], hi_r[h]);
        }
        uint32_t lo_all, hi_all;  // what every row of the block sees
        {
            uint32_t t;
            key_range(p, seq, i1, i1, lo_all, t);
            key_range(p, seq, i0, i0, t, hi_all);
        }
        const uint32_t edge_hi = min(hi_all, key1);
        constexpr uint32_t REFILL = TMA ? 2 : 1;  // tiles asked for where one has been read, until the ring is full
        // The next tile in the ring has arrived: its slot.
        auto arrived = [&](uint32_t &slot) {
            slot = at;
            if constexpr (TMA) {
                if (!__all_sync(0xffffffffu, q4k::mbar_wait(bars + 8 * at, (phases >> at) & 1u, abortp))) {
                    if (lane == 0) *abortp = 1, *(volatile uint32_t *)p.status = (32u << 24) | blockIdx.x;
                    return false;
                }
                phases ^= 1u << at;
            } else {
                cp_async_wait<SLOTS - 1>();
                __syncwarp();
            }
            if (++at == SLOTS) at = 0;
            return true;
        };
        for (uint32_t j = 0; j < mine; ++j) {
            const uint32_t key = key_of(j);
            uint32_t kt, vt;
            if (!arrived(kt)) break;
            uint32_t gone = 0;  // bit t: key t is not there
            if constexpr (TMA) {
                const uint32_t b = (holes >> (j % 16 * 2)) & 3u;
                gone = sp.box == 8 ? (b & 1u ? 0xffu : 0u) | (b & 2u ? 0xff00u : 0u) : b ? 0xffffu : 0u;
            } else if (row_hole) {
                const uint32_t k = key + (lane & 15u);
                gone = __ballot_sync(0xffffffffu, k < key1 && (uint32_t)__ldcg(table + p.page.div(k)) >= p.cache.num_pages) & 0xffffu;
            }
            float sc[2][4] = {}, odd[2][4] = {};  // two chains of MMAs for each eight keys
            const uint32_t ka = ring + kt * C::TILE;
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
                ldsm4(ka + piece_at((lane & 7u) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1u)), b);
                mma_bf16(k % 2 ? odd[0] : sc[0], a, b[0], b[1]);
                mma_bf16(k % 2 ? odd[1] : sc[1], a, b[2], b[3]);
            }
            __syncwarp();  // the tile is read
            ++done;
            feed(REFILL);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) sc[n][x] = (sc[n][x] + odd[n][x]) * p.scale_log2;
            const bool edge = key < lo_all || key + kStep > edge_hi;  // keys that not all rows see, or behind the sequence
            if (gone || edge) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const uint32_t t = 8 * n + 2 * (lane & 3u) + (x & 1);
                        if (((gone >> t) & 1u) || key + t < lo_r[x >> 1] || key + t >= min(hi_r[x >> 1], key1)) sc[n][x] = -INFINITY;
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
            if (!arrived(vt)) break;
            const uint32_t va = ring + vt * C::TILE;
            if (edge && ((TMA && key + kStep > seq.keys) || some_unseen(seq, key, kStep, lo_all, hi_all))) {
#pragma unroll 1
                for (uint32_t c = lane; c < kStep * (DP / 8); c += 32) {
                    const uint32_t k = key + c / (DP / 8), x = va + piece_at(c / (DP / 8), c % (DP / 8));
                    if (k >= seq.keys) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(x), "r"(0) : "memory");  // may hold anything: no values
                    else if (some_unseen(k, lo_all, hi_all) && make_finite<1>([&](int) { return x; })) *(volatile int *)&made_finite = 1;
                }
                if (TMA) fence_async_smem();  // the slot's next writer is the copy engine
                __syncwarp();
            }
#pragma unroll
            for (uint32_t n = 0; n < DP / 16; ++n) {
                uint32_t b[4];
                // keys 0-7, 8-15 of columns 16 n, then of 8 more
                ldsm4_t(va + piece_at(lane & 15u, 2 * n + (lane >> 4)), b);
                mma_bf16(o[2 * n], pf, b[0], b[1]);
                mma_bf16(o[2 * n + 1], pf, b[2], b[3]);
            }
            __syncwarp();  // the tile is read
            ++done;
            feed(REFILL);
        }
        if constexpr (TMA) {
            if (*abortp) {  // what is on its way must land before the block ends
                const long long t0 = clock64();
                for (uint32_t k = done; k < issued; ++k) {
                    const uint32_t slot = (to + SLOTS - (issued - k)) % SLOTS;
                    while (!q4k::mbar_try(bars + 8 * slot, (phases >> slot) & 1u))
                        if (clock64() - t0 > 20000000ll) break;
                }
            }
        } else {
            cp_async_wait<0>();
        }

        // ---- the warps meet: sums to the block's maximum, every warp's accumulators in its ring ----
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            if ((lane & 3u) == 0) ml[warp * ROWS + lane / 4 + 8 * h] = make_float2(m[h], l[h]);
        }
        __syncthreads();
        if (*abortp) return;  // of the whole block: no thread sets it between the barriers
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float t = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < C::WARPS; ++w) t = fmaxf(t, ml[w * ROWS + lane / 4 + 8 * h].x);
            const float f = m[h] == -INFINITY ? 0.0f : exp2_fast(m[h] - t);
            float *dst = reinterpret_cast<float *>(smem + warp * C::RING) + (lane / 4 + 8 * h) * DP;
#pragma unroll
            for (uint32_t n = 0; n < DP / 8; ++n)  // 16-byte pieces swizzled: eight rows on different banks
                *reinterpret_cast<float2 *>(dst + (((2 * n + ((lane >> 1) & 1u)) ^ (lane / 4)) << 2) + (lane & 1u) * 2) =
                    make_float2(o[n][2 * h] * f, o[n][2 * h + 1] * f);
        }
        __syncthreads();
        float *part = P::at(p.work, blockIdx.x, u0 == 0);
        for (uint32_t c = tid; c < min(ROWS, rows - row0) * (DP / 4); c += C::THREADS) {
            const uint32_t r = c / (DP / 4), x = c % (DP / 4);
            if (x * 4 >= d) continue;
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
        u += line.places(n_units);
        if (u >= u_end) break;
        L::next(p, cur);
        if (TMA) fence_async_smem();  // the rings' next writer is the copy engine
        __syncthreads();              // rings, Q and ml are read
    }
    __syncthreads();
    if (made_finite) {
        add_not_finite<DP, ROWS, UNIT, L>(p, shared, C::THREADS);
        __syncthreads();
    }
    finish_parts<DP, ROWS>(p, line, pending, has, C::THREADS, came, reinterpret_cast<float *>(smem), C::WARPS * C::RING / 4);
}

}  // namespace attn
}  // namespace tessl
