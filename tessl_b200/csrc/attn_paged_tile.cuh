// Attention of many rows per key head (prompts, chunks of them) over a paged cache, on the tcgen05 tensor cores.
//
// An item is NT tiles of 128 rows (tokens x the query heads of one key head) of a sequence; its keys come in tiles of 128.
// S = Q K^T of a tile is one MMA chain into TMEM, a thread of the softmax warpgroups has one row of it: running maximum and
// sum, weights rounded to bf16 and written back to TMEM over the scores, from where the second MMA chain takes them as its A operand
// and adds P V to the row tile's accumulators in TMEM. Heads of up to 128 columns: two row tiles, so that the tensor core works on
// one while the softmax of the other runs, and both read the same K and V. Wider heads: one row tile, whose accumulators take half of
// TMEM, and two buffers of scores.
//
// The accumulators are scaled when a row's maximum has grown by more than 2^8 since they were last, not with every new
// maximum (the divisor is scaled with them, so the quotient is the same; the weights stay below 2^8).
//
// K and V come by TMA, page by page, as 64-column chunks of 128 keys with the 128-byte swizzle: K is the K-major B operand of
// the first product, V the MN-major B operand of the second. Pages outside the cache and keys past the sequence's last page
// arrive as zeros; slots of the last page behind the sequence may hold anything, so their rows of V are zeroed in shared
// memory before the product (0 times NaN).
//
// Rounding of the weights: see attn_paged_split.cuh. A value of V that is not finite reaches the rows that see its token; in the tiles
// in which some rows see the token and others do not, it reaches those too (0 times it).
//
// Roles: warps 0 .. 4 NT - 1 softmax, Q and the results, one warp TMA, one warp TMEM and MMA issue. Every wait is bounded; on a
// timeout the status word is set and all roles fall through to the end.
#pragma once
#include "attn_paged_common.cuh"
#include "prefill_common.cuh"

namespace tessl {
namespace attn {

constexpr uint32_t kTileKeys = 128;

template <int DP>
struct TileCfg {
    static constexpr uint32_t NT = DP <= 128 ? 2 : 1;      // row tiles of an item
    static constexpr uint32_t NS = DP <= 128 ? 1 : 2;      // buffers of scores of a row tile
    static constexpr uint32_t ROWS = NT * 128;
    static constexpr uint32_t CHUNKS = DP / 64;            // 64-column chunks of a row
    static constexpr uint32_t CPS = DP == 256 ? 2 : CHUNKS;  // chunks per slot of the ring
    static constexpr uint32_t SPT = CHUNKS / CPS;          // slots per tile of K or V
    static constexpr uint32_t CHUNK = 128 * 128, SLOT = CPS * CHUNK;  // bytes
    static constexpr uint32_t Q_BYTES = NT * CHUNKS * CHUNK;
    static constexpr uint32_t SLOTS = DP == 64 ? 11 : DP == 192 ? 3 : 5;
    static constexpr uint32_t BARS_T = 4 * NS + 2, NBARS = 2 * SLOTS + NT * BARS_T + 1;
    static constexpr uint32_t SMEM = Q_BYTES + SLOTS * SLOT + NBARS * 8 + 1024;  // + slack to align the base to 1 KiB
    // Two softmax warpgroups: a third one of the TMA and the MMA warp (and two that do nothing) gives them registers, 168 a
    // thread at launch: 8 x 208 + 4 x 88 = 12 x 168.
    static constexpr bool REGS = NT == 2;
    static constexpr uint32_t SOFTMAX_WARPS = 4 * NT, THREADS = (SOFTMAX_WARPS + (REGS ? 4 : 2)) * 32;
    static constexpr uint32_t POLY = NT == 2 ? 4 : 0;      // of 16 pairs of weights: 2^x by polynomial
    static constexpr uint32_t S_COL = 256;                 // TMEM columns: accumulators from 0, scores from here
    static_assert(SMEM <= 227 * 1024 - 64, "shared memory");
    static_assert(sizeof(typename Line<ROWS, kTileKeys, THREADS>::Shared) <= SLOTS * SLOT, "the scan of the line uses the ring");
    static_assert(SMEM > 227 * 1024 / 2, "two blocks on an SM would both want all of its TMEM");
};

struct TileParams {
    Params p;
    uint32_t box;      // tokens per TMA box
    uint32_t negate;   // the scale is negative: the first product's A operand is negated instead
};

/// Box of the cache: 64 columns of one key head, `box` tokens of one page.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
        "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
/// D[tmem] (+)= A[tmem] . B[smem] for one K = 16 slice.
__device__ __forceinline__ void tcgen05_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
/// Descriptor of 64-column chunks of V, MN-major: 128-byte rows (64 columns of one key), groups of eight keys 1024 B apart, chunks
/// of 64 columns CHUNK bytes apart.
__device__ __forceinline__ uint64_t v_desc(uint32_t smem_addr, uint32_t chunk)
{
    return (uint64_t)((smem_addr & 0x3ffffu) >> 4) | ((uint64_t)(chunk >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
#define TMEM_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
/// Load and wait in one statement (see pf::tmem_ld32).
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,"
        "%25,%26,%27,%28,%29,%30,%31,%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,%48,%49,%50,%51,%52,%53,%54,%55,%56,"
        "%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : TMEM_R8(r, 0), TMEM_R8(r, 8), TMEM_R8(r, 16), TMEM_R8(r, 24), TMEM_R8(r, 32), TMEM_R8(r, 40), TMEM_R8(r, 48), TMEM_R8(r, 56)
        : "r"(taddr));
}
#undef TMEM_R8
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ uint64_t f32_pair(float lo, float hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f32_unpair(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
/// The larger, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
/// 2^x of two finite values on the FMA pipe: x = n + f with n the nearest integer (Cody and Waite), 2^f by the polynomial of degree 4
/// with the least relative error on [-1/2, 1/2] (Remez; 2.7e-6 in f32), n added to the exponent. Below 2^-126: 2^-126.
__device__ __forceinline__ uint64_t exp2_poly(uint64_t x)
{
    float a, b;
    f32_unpair(x, a, b);
    x = f32_pair(fmaxf(a, -126.0f), fmaxf(b, -126.0f));
    constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: the sum's low bits are n
    const uint64_t n = add2(x, f32_pair(kRound, kRound));
    const uint64_t f = add2(x, fma2(n, f32_pair(-1.0f, -1.0f), f32_pair(kRound, kRound)));
    uint64_t y = fma2(f, f32_pair(0.009570102207362652f, 0.009570102207362652f), f32_pair(0.05591785907745361f, 0.05591785907745361f));
    y = fma2(y, f, f32_pair(0.240247443318367f, 0.240247443318367f));
    y = fma2(y, f, f32_pair(0.6931217908859253f, 0.6931217908859253f));
    y = fma2(y, f, f32_pair(0.9999992847442627f, 0.9999992847442627f));
    float na, nb, ya, yb;
    f32_unpair(n, na, nb), f32_unpair(y, ya, yb);
    return f32_pair(__uint_as_float(__float_as_uint(ya) + (__float_as_uint(na) << 23)), __uint_as_float(__float_as_uint(yb) + (__float_as_uint(nb) << 23)));
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int DP>
__global__ void __launch_bounds__(TileCfg<DP>::THREADS, 1)
    attn_paged_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TileParams tp)
{
    using C = TileCfg<DP>;
    using L = Line<C::ROWS, kTileKeys, C::THREADS>;
    using P = Part<C::ROWS, DP>;
    using q4k::mbar_arrive;
    using q4k::mbar_expect_tx;
    using q4k::mbar_init;
    using q4k::mbar_try;
    using q4k::mbar_wait;
    constexpr uint32_t NT = C::NT, NS = C::NS;
    asm volatile("griddepcontrol.launch_dependents;");
    const Params &p = tp.p;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const uint32_t base = (q4k::smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_smem = base, ring = base + C::Q_BYTES, bar0 = ring + C::SLOTS * C::SLOT;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    auto slot_full = [&](uint32_t s) { return bar0 + 8 * s; };
    auto slot_empty = [&](uint32_t s) { return bar0 + 8 * (C::SLOTS + s); };
    const uint32_t bar1 = bar0 + 16 * C::SLOTS;
    auto s_full = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + b); };           // scores are there
    auto p_full = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + NS + b); };      // weights are there, scores read
    // A product with V is done. One for each buffer of scores: products i and i + 1 may both be under way, i + 2 starts behind i's end.
    auto o_full = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + 2 * NS + b); };
    auto p_half = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + 3 * NS + b); };  // weights of the first 64 keys
    auto q_full = [&](uint32_t t) { return bar1 + 8 * (t * C::BARS_T + 4 * NS); };
    auto o_free = [&](uint32_t t) { return bar1 + 8 * (t * C::BARS_T + 4 * NS + 1); };              // the item's result is read
    const uint32_t done = bar1 + 8 * (NT * C::BARS_T);

    if (warp == 0) {
        if (lane < C::SLOTS) mbar_init(slot_full(lane), 1), mbar_init(slot_empty(lane), 1);
        if (lane < NT) {
            for (uint32_t b = 0; b < NS; ++b) mbar_init(s_full(lane, b), 1), mbar_init(p_full(lane, b), 4), mbar_init(o_full(lane, b), 1), mbar_init(p_half(lane, b), 4);
            mbar_init(q_full(lane), 4), mbar_init(o_free(lane), 4);
        }
        if (lane == 0) {
            abort_flag = 0;
            mbar_init(done, 1);
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::SOFTMAX_WARPS + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(q4k::smem_u32(&tmem_slot)), "r"(pf::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pf::tcgen05_fence_before();
    __syncthreads();
    pf::tcgen05_fence_after();
    const uint32_t tmem = tmem_slot;
    volatile int *abortp = &abort_flag;
    auto fail = [&](uint32_t role, uint32_t where) {
        *abortp = 1;
        *(volatile uint32_t *)p.status = (role << 24) | (where & 0xffffffu);
    };
    asm volatile("griddepcontrol.wait;" ::: "memory");

    L line;
    Cursor cur;
    uint64_t u = 0, u_end = 0;
    if (line.start(p, blockIdx.x, *reinterpret_cast<typename L::Shared *>(smem_raw + (ring - q4k::smem_u32(smem_raw))), u, cur))
        u_end = line.cut(blockIdx.x + 1);
    fence_async_smem();  // the ring's next writer is the copy engine
    __syncthreads();
    // The item at the cursor, as every role sees it: tiles of keys k0, k0 + 128, ...
    uint32_t n_units, n, k0, row0, rows;
    auto item = [&] {
        n_units = (uint32_t)min((uint64_t)(cur.units - cur.u0), u_end - u);
        rows = cur.seq.news * p.group, row0 = cur.block * C::ROWS;
        uint32_t lo, hi;
        key_range(p, cur.seq, row0 / p.group, (min(row0 + C::ROWS, rows) - 1) / p.group, lo, hi);
        k0 = (cur.first + cur.u0) * kTileKeys;
        const uint32_t k1 = min(k0 + n_units * kTileKeys, hi);
        n = k1 > k0 ? (k1 - k0 + kTileKeys - 1) / kTileKeys : 0;
    };
    // Tiles are loaded and used in the order K_0 .. K_(NS-1), V_0, K_NS, V_1, ...: where among the item's K_j and V_j are.
    auto k_place = [&](uint32_t j) { return j < NS ? j : 2 * j - NS + 1; };
    auto v_place = [&](uint32_t j) { return j + min(n, j + NS); };
    uint32_t tiles = 0;  // of K and V, in front of the item

    // Within its branch each, where the compiler can tell what holds.
    auto fewer_regs = [] {
        if constexpr (C::REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    };
    if (warp == C::SOFTMAX_WARPS) {
        // ------------------------------------------------ TMA ---
        fewer_regs();
        const uint32_t boxes = kTileKeys / tp.box;
        uint32_t at = 0, phase = 0, issued = 0;  // ring position
        auto load = [&](const CUtensorMap *map, int page, int slot) -> bool {
            for (uint32_t i = 0; i < C::SPT; ++i) {
                bool ok = true;
                if (lane == 0) {
                    ok = mbar_wait(slot_empty(at), phase ^ 1u, abortp, 20);
                    if (!ok) fail(1, issued);
                    if (ok) mbar_expect_tx(slot_full(at), C::SLOT);
                }
                if (!__shfl_sync(0xffffffffu, (int)ok, 0)) return false;
                if (lane < boxes)
                    for (uint32_t c = 0; c < C::CPS; ++c)
                        tma_load_4d(ring + at * C::SLOT + c * C::CHUNK + lane * tp.box * 128, map, (int)((i * C::CPS + c) * 64), (int)cur.kv_head, slot, page,
                                    slot_full(at));
                __syncwarp();
                ++issued;
                if (++at == C::SLOTS) at = 0, phase ^= 1u;
            }
            return true;
        };
        bool ok = true;
        asm volatile("fence.proxy.async.global;" ::: "memory");  // ordinary stores of the launch in front, read by the copy engine
        while (u < u_end && ok) {
            item();
            const int32_t *table = p.seqs.table + (size_t)cur.seq.index * p.seqs.max_pages;
            // Lane l's box of tile j: keys k0 + 128 j + l box ..; past the sequence a page that is not there.
            auto find = [&](uint32_t j, int &page, int &slot) {
                const uint32_t key = k0 + j * kTileKeys + lane * tp.box;
                page = (int)p.cache.num_pages, slot = 0;
                if (j < n && lane < boxes && key < cur.seq.keys) {
                    const uint32_t pg = (uint32_t)__ldcg(table + key / p.cache.page_size);
                    if (pg < p.cache.num_pages) page = (int)pg, slot = (int)(key % p.cache.page_size);
                }
            };
            int pk[NS + 1], sk[NS + 1];  // pages of tiles j .. j + NS
            for (uint32_t j = 0; j < NS; ++j) {
                find(j, pk[j], sk[j]);
                if (j < n && ok) ok = load(&map_k, pk[j], sk[j]);
            }
            find(NS, pk[NS], sk[NS]);
            for (uint32_t j = 0; j < n && ok; ++j) {
                int np, ns;
                find(j + NS + 1, np, ns);
                ok = load(&map_v, pk[0], sk[0]);
                if (ok && j + NS < n) ok = load(&map_k, pk[NS], sk[NS]);
#pragma unroll
                for (uint32_t i = 0; i < NS; ++i) pk[i] = pk[i + 1], sk[i] = sk[i + 1];
                pk[NS] = np, sk[NS] = ns;
            }
            u += n_units;
            if (u < u_end) L::next(p, cur);
        }
        if (*abortp && lane == 0) {  // what is on its way must land before the block ends
            const long long t0 = clock64();
            for (uint32_t i = issued > C::SLOTS ? issued - C::SLOTS : 0; i < issued; ++i)
                while (!mbar_try(slot_full(i % C::SLOTS), (i / C::SLOTS) & 1u))
                    if (clock64() - t0 > 20000000ll) break;
        }
        __syncwarp();
    } else if (warp == C::SOFTMAX_WARPS + 1) {
        // ------------------------------------------------ MMA ---
        fewer_regs();
        if (lane == 0) {
            constexpr uint32_t kBf16 = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // f32 += bf16 . bf16, M = 128
            const uint32_t idesc_qk = kBf16 | ((kTileKeys >> 3) << 17) | (tp.negate << 13);  // -A
            constexpr uint32_t idesc_pv = kBf16 | (1u << 16) | ((C::CPS * 64 >> 3) << 17);
            uint32_t used[NT], items[NT];  // tiles of scores, items of each row tile
            for (uint32_t t = 0; t < NT; ++t) used[t] = 0, items[t] = 0;
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity, uint32_t role) {
                if (ok && !mbar_wait(bar, parity, abortp)) ok = false, fail(role, tiles);
                return ok;
            };
            auto wait_slots = [&](uint32_t place) {  // of a tile
                for (uint32_t i = 0; i < C::SPT; ++i) {
                    const uint32_t x = (tiles + place) * C::SPT + i;
                    wait(slot_full(x % C::SLOTS), (x / C::SLOTS) & 1u, 2);
                }
            };
            while (u < u_end && ok) {
                item();
                const uint32_t live = rows - row0 > 128 ? NT : 1;
                auto scores = [&](uint32_t t, uint32_t j) {
                    const uint32_t buf = (used[t] + j) % NS, place = k_place(j);
                    const uint32_t dst = tmem + C::S_COL + (t * NS + buf) * 128;
#pragma unroll
                    for (uint32_t c = 0; c < C::CHUNKS; ++c) {
                        const uint32_t x = ((tiles + place) * C::SPT + c / C::CPS) % C::SLOTS;
                        const uint64_t a = pf::umma_desc(q_smem + (t * C::CHUNKS + c) * C::CHUNK);
                        const uint64_t b = pf::umma_desc(ring + x * C::SLOT + (c % C::CPS) * C::CHUNK);
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) pf::tcgen05_mma_f16(dst, a + 2 * k, b + 2 * k, idesc_qk, c || k);
                        if ((c + 1) % C::CPS == 0 && t + 1 == live) pf::tcgen05_commit(slot_empty(x));
                    }
                    pf::tcgen05_commit(s_full(t, buf));
                };
                for (uint32_t j = 0; j < NS && j < n && ok; ++j) {
                    wait_slots(k_place(j));
                    for (uint32_t t = 0; t < live && ok; ++t) {
                        if (j == 0 && !wait(q_full(t), items[t] & 1u, 3)) break;
                        pf::tcgen05_fence_after();
                        scores(t, j);
                    }
                }
                for (uint32_t j = 0; j < n && ok; ++j) {
                    for (uint32_t t = 0; t < live; ++t) {
                        const uint32_t i = used[t] + j, buf = i % NS;
                        if (!wait(p_half(t, buf), (i / NS) & 1u, 4)) break;
                        if (j == 0 && items[t] && !wait(o_free(t), (items[t] - 1) & 1u, 5)) break;
                        if (t == 0) wait_slots(v_place(j));
                        if (!ok) break;
                        pf::tcgen05_fence_after();
                        const uint32_t a = tmem + C::S_COL + (t * NS + buf) * 128, place = v_place(j);
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {  // the two halves of the keys
                            if (h == 1) {
                                if (!wait(p_full(t, buf), (i / NS) & 1u, 11)) break;
                                pf::tcgen05_fence_after();
                            }
#pragma unroll
                            for (uint32_t s = 0; s < C::SPT; ++s) {
                                const uint32_t x = ((tiles + place) * C::SPT + s) % C::SLOTS;
                                const uint64_t b = v_desc(ring + x * C::SLOT, C::CHUNK);
#pragma unroll
                                for (uint32_t k = h * kTileKeys / 32; k < (h + 1) * kTileKeys / 32; ++k)
                                    tcgen05_mma_ts(tmem + t * DP + s * C::CPS * 64, a + 8 * k, b + k * (2048 >> 4), idesc_pv, j || k);
                                if (h == 1 && t + 1 == live) pf::tcgen05_commit(slot_empty(x));
                            }
                        }
                        if (!ok) break;
                        if (NS > 1 || j + 1 == n) pf::tcgen05_commit(o_full(t, buf));
                        if (j + NS < n) {
                            if (t == 0) wait_slots(k_place(j + NS));
                            if (!ok) break;
                            pf::tcgen05_fence_after();
                            scores(t, j + NS);
                        }
                    }
                }
                for (uint32_t t = 0; t < live && n; ++t) used[t] += n, ++items[t];
                tiles += 2 * n;
                u += n_units;
                if (u < u_end) L::next(p, cur);
            }
            // Also after an abort: nothing may still read shared memory or TMEM when the block ends.
            pf::tcgen05_commit(done);
            const long long t0 = clock64();
            while (!mbar_try(done, 0u))
                if (clock64() - t0 > 4000000000ll) break;
        }
        __syncwarp();
    } else if (warp < C::SOFTMAX_WARPS) {
        // ------------------------------------------------ softmax ---
        if constexpr (C::REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const uint32_t t = warp >> 2, r = tid & 127;                     // row tile, row
        const uint32_t lanes = (warp & 3u) << 21;                        // this warp's quarter of the TMEM lanes
        const uint32_t o_tmem = tmem + lanes + t * DP, d = p.cache.head_dim;
        const float c2 = p.scale_log2;
        const uint64_t c2x2 = f32_pair(c2, c2);
        uint32_t used = 0, items = 0;
        bool ok = true;
        // A whole warp's wait: every lane waits, all go on or none.
        auto wait = [&](uint32_t bar, uint32_t parity, uint32_t role, uint32_t where) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abortp));
            if (!ok && lane == 0) fail(role, where);
            return ok;
        };
        auto live = [&] { return u < u_end && row0 + t * 128 < rows; };  // the item at the cursor has rows here
        // Q of the item at the cursor. The scores of the one before have been read, so nothing reads its Q any more.
        auto load_q = [&] {
            if (!live() || n == 0) return;
            for (uint32_t i = r; i < 128 * (DP / 8); i += 128) {
                const uint32_t qr = i / (DP / 8), cc = i % (DP / 8), row = row0 + t * 128 + qr;
                const bool there = row < rows && cc * 8 < d;
                uint32_t token = 0, head = 0;
                if (there) row_at(p, cur.seq, cur.kv_head, row, token, head);
                const uint32_t dst = q_smem + (t * C::CHUNKS + cc / 8) * C::CHUNK + qr * 128 + (((cc & 7u) ^ (qr & 7u)) << 4);
                cp_async16(dst, p.q + (there ? (size_t)token * p.q_stride + (size_t)head * d + cc * 8 : 0), there);
            }
            cp_async_commit();
        };
        auto q_ready = [&] {
            if (!live() || n == 0) return;
            cp_async_wait<0>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(t));
        };
        if (u < u_end) item();
        load_q();
        q_ready();
        while (u < u_end) {
            const bool mine = live();
            const uint32_t row = row0 + t * 128 + r, tiles_n = n;
            float top = -INFINITY, sum = 0.0f;  // raw score that the weights refer to; of the weights
            uint16_t *out = nullptr;
            if (mine) {
                uint32_t lo_r, hi_r;  // rows past the last see what that sees
                {
                    const uint32_t i = min(row, rows - 1) / p.group;
                    key_range(p, cur.seq, i, i, lo_r, hi_r);
                }
                const uint32_t lo_all = __shfl_sync(0xffffffffu, lo_r, 31), hi_all = __shfl_sync(0xffffffffu, hi_r, 0);
                const int32_t *table = p.seqs.table + (size_t)cur.seq.index * p.seqs.max_pages;
                auto missing = [&](uint32_t j) {  // lane l: the page of keys 4 l .. 4 l + 3 of tile j is not there
                    const uint32_t key = k0 + j * kTileKeys + 4 * lane;
                    return j < n && key < cur.seq.keys && (uint32_t)__ldcg(table + key / p.cache.page_size) >= p.cache.num_pages;
                };
                bool hole = missing(0);
                for (uint32_t j = 0; j < n; ++j) {
                    const uint32_t buf = (used + j) % NS, key = k0 + j * kTileKeys;
                    const uint32_t s_tmem = tmem + lanes + C::S_COL + (t * NS + buf) * 128;
                    const uint32_t holes = __ballot_sync(0xffffffffu, hole);
                    hole = missing(j + 1);
                    if (!wait(s_full(t, buf), ((used + j) / NS) & 1u, 6, j)) break;
                    pf::tcgen05_fence_after();
                    uint32_t s[2][64];
                    tmem_ld64(s_tmem, s[0]);
                    tmem_ld64(s_tmem + 64, s[1]);
                    const bool masked = holes || key < lo_all || key + kTileKeys > hi_all;
                    if (masked) {
#pragma unroll
                        for (uint32_t x = 0; x < 128; ++x)
                            if (key + x < lo_r || key + x >= hi_r || ((holes >> (x / 4)) & 1u)) s[x / 64][x % 64] = 0xff800000u;
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (uint32_t x = 0; x < 128; x += 8)
#pragma unroll
                        for (uint32_t y = 0; y < 4; ++y)
                            m4[y] = max_nan(m4[y], max_nan(__uint_as_float(s[x / 64][x % 64 + 2 * y]), __uint_as_float(s[x / 64][x % 64 + 2 * y + 1])));
                    const float m = max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3]));
                    const bool grow = (m - top) * c2 > 8.0f;  // never where both are -inf, or m is NaN
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? exp2_fast((top - m) * c2) : 1.0f;
                        if (__any_sync(0xffffffffu, grow && top != -INFINITY)) {
                            // With one buffer the scores came behind the last product with V; with two, that may still run.
                            if (NS > 1 && !wait(o_full(t, (used + j - 1) % NS), ((used + j - 1) / NS) & 1u, 7, j)) break;
                            pf::tcgen05_fence_after();
#pragma unroll 1
                            for (uint32_t x = 0; x < DP; x += 32) {
                                uint32_t o[32];
                                pf::tmem_ld32(o_tmem + x, o);
#pragma unroll
                                for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
                                tmem_store32(o_tmem + x, o);
                            }
                        }
                        if (grow) sum *= f, top = m;
                    }
                    if (key + kTileKeys > cur.seq.keys) {  // slots behind the sequence: no values
                        for (uint32_t i = 0; i < C::SPT; ++i) {
                            const uint32_t x = (tiles + v_place(j)) * C::SPT + i, slot = ring + x % C::SLOTS * C::SLOT;
                            if (!wait(slot_full(x % C::SLOTS), (x / C::SLOTS) & 1u, 8, j)) break;
                            if (key + r >= cur.seq.keys)
                                for (uint32_t y = 0; y < C::CPS * 8; ++y)
                                    asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(slot + y / 8 * C::CHUNK + r * 128 + (y % 8) * 16), "r"(0) : "memory");
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (!ok) break;
                    }
                    const float off = top == -INFINITY ? 0.0f : -top * c2;
                    const uint64_t offx2 = f32_pair(off, off);
                    // The polynomial knows neither infinities nor NaN: rows with any, and masked tiles, do without it.
                    const bool plain = masked || __any_sync(0xffffffffu, !(m < INFINITY) || top == -INFINITY);
                    uint64_t s2[2] = {0, 0};
                    auto half = [&](uint32_t h, auto poly) {
                        uint32_t w[32];
#pragma unroll
                        for (uint32_t x = 0; x < 32; ++x) {
                            const uint64_t y = fma2(f32_pair(__uint_as_float(s[h][2 * x]), __uint_as_float(s[h][2 * x + 1])), c2x2, offx2);
                            uint64_t e;
                            if (decltype(poly)::value && (int)(x % 16) < (int)C::POLY) {
                                e = exp2_poly(y);
                            } else {
                                float a, b;
                                f32_unpair(y, a, b);
                                e = f32_pair(exp2_fast(a), exp2_fast(b));
                            }
                            s2[x & 1] = add2(s2[x & 1], e);
                            float a, b;
                            f32_unpair(e, a, b);
                            w[x] = bf16_pair(a, b);
                        }
                        tmem_store32(s_tmem + h * 32, w);
                        tmem_store_wait();
                        pf::tcgen05_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(h == 0 ? p_half(t, buf) : p_full(t, buf));
                    };
                    if (plain || C::POLY == 0) {
                        half(0, std::false_type{}), half(1, std::false_type{});
                    } else {
                        half(0, std::true_type{}), half(1, std::true_type{});
                    }
                    float a, b;
                    f32_unpair(add2(s2[0], s2[1]), a, b);
                    sum += a + b;
                }
                if (!ok) break;
                used += n;
                if (row < rows) {
                    uint32_t token, head;
                    row_at(p, cur.seq, cur.kv_head, row, token, head);
                    out = p.out + ((size_t)token * p.n_heads + head) * d;
                }
            }
            const bool whole = n_units == cur.units;
            float *part = P::at(p.work, blockIdx.x, cur.u0 == 0);
            tiles += 2 * n;
            u += n_units;
            if (u < u_end) L::next(p, cur), item();
            load_q();  // of the next item, while the last product runs
            if (mine && tiles_n) {
                const uint32_t last = used - 1;
                if (!wait(o_full(t, last % NS), (NS > 1 ? last / NS : items) & 1u, 9, 0)) break;
                pf::tcgen05_fence_after();
                ++items;
            }
            q_ready();
            if (!mine) continue;
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll 1
            for (uint32_t x = 0; x < DP; x += 32) {
                if (x >= d) break;
                uint32_t o[32];
                if (tiles_n) {
                    pf::tmem_ld32(o_tmem + x, o);
                } else {
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = 0;
                }
                if (out && whole) {
#pragma unroll
                    for (uint32_t y = 0; y < 32; y += 8) {
                        if (x + y >= d) break;
                        uint4 v;
                        v.x = bf16_pair(__uint_as_float(o[y]) * inv, __uint_as_float(o[y + 1]) * inv);
                        v.y = bf16_pair(__uint_as_float(o[y + 2]) * inv, __uint_as_float(o[y + 3]) * inv);
                        v.z = bf16_pair(__uint_as_float(o[y + 4]) * inv, __uint_as_float(o[y + 5]) * inv);
                        v.w = bf16_pair(__uint_as_float(o[y + 6]) * inv, __uint_as_float(o[y + 7]) * inv);
                        *reinterpret_cast<uint4 *>(out + x + y) = v;
                    }
                } else if (out) {
#pragma unroll
                    for (uint32_t y = 0; y < 32; y += 4)
                        *reinterpret_cast<uint4 *>(part + P::four(t * 128 + r, (x + y) / 4)) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
                }
                __syncwarp();
            }
            if (!whole && out) part[P::TOP + t * 128 + r] = top == -INFINITY ? top : top * c2, part[P::SUM + t * 128 + r] = sum;
            if (tiles_n) {
                pf::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_free(t));
            }
        }
        __syncwarp();
    } else {
        fewer_regs();
    }
    pf::tcgen05_fence_before();
    __syncthreads();
    if (warp == C::SOFTMAX_WARPS + 1) {
        pf::tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(pf::kTmemCols) : "memory");
    }
}

}  // namespace attn
}  // namespace tessl
