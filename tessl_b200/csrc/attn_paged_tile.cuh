// Attention of many rows per key head (prompts, chunks of them) over a paged cache, on the tcgen05 tensor cores.
//
// An item is NT tiles of 128 rows (tokens x the query heads of one key head) of a sequence; its keys come in tiles of 128.
// S = Q K^T of a step of keys is one MMA chain into TMEM; a softmax thread has 64 keys of a row of it: running maximum and sum,
// weights rounded to bf16 and written back to TMEM over the scores, from where the second MMA chain takes them as its A operand
// and adds P V to the row tile's accumulators in TMEM. Two buffers of scores for each row tile: the first chain is a step ahead.
// Heads of up to 128 columns: two row tiles that read the same K and V, steps of 64 keys. Wider heads: one row tile, whose
// accumulators take half of TMEM, steps of 128 keys, two threads for a row.
//
// The accumulators are scaled when a row's maximum has grown by more than 2^8 since they were last, not with every new
// maximum (the divisor is scaled with them, so the quotient is the same; the weights stay below 2^8).
//
// K and V come by TMA, page by page, as 64-column chunks of 128 keys with the 128-byte swizzle: K is the K-major B operand of
// the first product, V the MN-major B operand of the second. Pages outside the cache and keys past the sequence's last page
// arrive as zeros; slots of the last page behind the sequence may hold anything, so their rows of V are zeroed in shared
// memory before the product (0 times NaN), as are values of V that are not finite and that some rows see and others do not.
//
// Rounding of the weights: see attn_paged_split.cuh.
//
// Bound by the chain scores, softmax, weights, product of a step, of which a row tile has two under way: 1024 tokens over 33024 keys, 32
// heads of 128 on 8, take 615 us call behind call (888 TFLOP/s, of 1382 for a library product that runs as long: both at the power cap, this
// at 1570 MHz) and 529 us in the first calls after a pause (1030 of 1668, at 1965 MHz); a prompt of 4096 with 16 heads of 256 on 4 215 us (639
// TFLOP/s): wide heads have one row tile, with two threads for a row that wait for each other's maxima.
//
// Roles: eight warps softmax, Q and the results, one warp TMA, a warp for each row tile MMA issue. Every wait is bounded; on a
// timeout the status word is set and all roles fall through to the end.
#pragma once
#include "attn_paged_split.cuh"
#include "prefill_common.cuh"

namespace tessl {
namespace attn {

constexpr uint32_t kTileKeys = 128;
// What a second part of an item costs, in tiles of keys: nine chunks of up to 300 tokens with a window of 1024 took 58 us with 12 and 78 us
// with 6, with up to 200 tokens over up to 1500 keys 33 us with 3 and more and 63 us with 0.
constexpr uint32_t kTileExtra = 12;

template <int DP>
struct TileCfg {
    static constexpr uint32_t NT = DP <= 128 ? 2 : 1;      // row tiles of an item
    static constexpr uint32_t TPR = 2 / NT;                // threads of a row
    static constexpr uint32_t SK = 64 * TPR;               // keys of a step
    static constexpr uint32_t NS = 2;                      // buffers of scores of a row tile
    static constexpr uint32_t SPK = kTileKeys / SK;        // steps per tile of keys
    static constexpr uint32_t AHEAD = NS / SPK;            // tiles of K in front of V
    static constexpr uint32_t ROWS = NT * 128;
    static constexpr uint32_t CHUNKS = DP / 64;            // 64-column chunks of a row
    static constexpr uint32_t CPS = DP == 256 ? 2 : CHUNKS;  // chunks per slot of the ring
    static constexpr uint32_t SPT = CHUNKS / CPS;          // slots per tile of K or V
    static constexpr uint32_t CHUNK = 128 * 128, SLOT = CPS * CHUNK;  // bytes
    static constexpr uint32_t Q_BYTES = NT * CHUNKS * CHUNK;
    static constexpr uint32_t SLOTS = DP == 64 ? 11 : DP == 192 ? 3 : 5;
    static constexpr uint32_t BARS_T = 3 * NS + 2, NBARS = 2 * SLOTS + NT * BARS_T + 1;
    static constexpr uint32_t X_BYTES = TPR == 2 ? NS * 2 * 128 * 4 : 0;  // what the two threads of a row tell each other
    static constexpr uint32_t SMEM = Q_BYTES + SLOTS * SLOT + X_BYTES + NBARS * 8 + 2 * sizeof(Pending) + 32;
    static constexpr uint32_t TMA_WARP = 4 * NT * TPR, MMA_WARP = TMA_WARP + 1, THREADS = (MMA_WARP + NT) * 32;
    static constexpr uint32_t S_COL = 256;                 // TMEM columns: accumulators from 0, scores from here
    static_assert(SMEM <= 227 * 1024, "shared memory");    // none of it static: the dynamic part starts at a multiple of 1 KiB
    static_assert(sizeof(typename Line<ROWS, kTileKeys, THREADS, kTileExtra>::Shared) <= SLOTS * SLOT, "the scan of the line uses the ring");
    static_assert(SMEM > 227 * 1024 / 2, "two blocks on an SM would both want all of its TMEM");
};

struct TileParams {
    Params p;
    uint32_t box;      // tokens per TMA box
    uint32_t negate;   // the scale is negative: the first product's A operand is negated instead
};

// A converged warp issues the MMAs, one election for four of them: descriptors stay warp-uniform values. (From a branch of one lane
// 16 MMAs took ~1500 clocks to issue, three times as long as to run.)
/// D[tmem] (+)= A[smem] . B[smem]^T, K = 64: two 64-column chunks, K-major, by the low words of their descriptors.
__device__ __forceinline__ void mma_ss4_elect(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u32 x1, %1, 2;\n\tadd.u32 x2, %1, 4;\n\tadd.u32 x3, %1, 6;\n\t"
        "add.u32 y1, %2, 2;\n\tadd.u32 y2, %2, 4;\n\tadd.u32 y3, %2, 6;\n\t"
        "mov.b64 a0, {%1, %5};\n\tmov.b64 a1, {x1, %5};\n\tmov.b64 a2, {x2, %5};\n\tmov.b64 a3, {x3, %5};\n\t"
        "mov.b64 b0, {%2, %5};\n\tmov.b64 b1, {y1, %5};\n\tmov.b64 b2, {y2, %5};\n\tmov.b64 b3, {y3, %5};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, 1;\n\t}" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(pf::kUmmaDescHi)
        : "memory");
}
/// D[tmem] (+)= A[tmem] . B[smem], K = 64: weights of 64 keys and their rows of V, MN-major (v_desc_lo).
__device__ __forceinline__ void mma_ts4_elect(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 b0, b1, b2, b3;\n\t.reg .b32 x1, x2, x3, y1, y2, y3;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u32 x1, %1, 8;\n\tadd.u32 x2, %1, 16;\n\tadd.u32 x3, %1, 24;\n\t"
        "add.u32 y1, %2, 128;\n\tadd.u32 y2, %2, 256;\n\tadd.u32 y3, %2, 384;\n\t"
        "mov.b64 b0, {%2, %5};\n\tmov.b64 b1, {y1, %5};\n\tmov.b64 b2, {y2, %5};\n\tmov.b64 b3, {y3, %5};\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b0, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x1], b1, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x2], b2, %3, 1;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x3], b3, %3, 1;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(pf::kUmmaDescHi)
        : "memory");
}
__device__ __forceinline__ void commit_elect(uint32_t bar)
{
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}
/// Low word of the descriptor of 64-column chunks of V, MN-major: 128-byte rows (64 columns of one key), groups of eight keys 1024 B
/// apart, chunks of 64 columns `chunk` bytes apart. The high word is that of the K-major tiles.
__device__ __forceinline__ uint32_t v_desc_lo(uint32_t smem_addr, uint32_t chunk) { return ((smem_addr & 0x3ffffu) >> 4) | ((chunk >> 4) << 16); }
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
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
        "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15])
        : "memory");
}
/// Load and wait in one statement (see pf::tmem_ld32).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
          "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
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
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

template <int DP>
__global__ void __launch_bounds__(TileCfg<DP>::THREADS, 1)
    attn_paged_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TileParams tp)
{
    using C = TileCfg<DP>;
    using L = Line<C::ROWS, kTileKeys, C::THREADS, kTileExtra>;
    using P = Part<C::ROWS, DP>;
    using q4k::mbar_arrive;
    using q4k::mbar_expect_tx;
    using q4k::mbar_init;
    using q4k::mbar_try;
    using q4k::mbar_wait;
    constexpr uint32_t NT = C::NT, NS = C::NS;
    asm volatile("griddepcontrol.launch_dependents;");
    const Params &p = tp.p;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t q_smem = q4k::smem_u32(smem_raw), ring = q_smem + C::Q_BYTES, bar0 = ring + C::SLOTS * C::SLOT + C::X_BYTES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem_raw + C::SMEM - 32);
    volatile int *abortp = reinterpret_cast<volatile int *>(smem_raw + C::SMEM - 24);
    volatile int *made_finite = reinterpret_cast<volatile int *>(smem_raw + C::SMEM - 20);
    Pending *pending = reinterpret_cast<Pending *>(smem_raw + C::SMEM - 32 - 2 * sizeof(Pending));  // items of which this block has a part
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    auto slot_full = [&](uint32_t s) { return bar0 + 8 * s; };
    auto slot_empty = [&](uint32_t s) { return bar0 + 8 * (C::SLOTS + s); };
    const uint32_t bar1 = bar0 + 16 * C::SLOTS;
    auto s_full = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + b); };           // scores are there
    auto p_full = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + NS + b); };      // weights are there, scores read
    auto o_full = [&](uint32_t t, uint32_t b) { return bar1 + 8 * (t * C::BARS_T + 2 * NS + b); };  // one of an item's last two products with V is done
    auto q_full = [&](uint32_t t) { return bar1 + 8 * (t * C::BARS_T + 3 * NS); };
    auto o_free = [&](uint32_t t) { return bar1 + 8 * (t * C::BARS_T + 3 * NS + 1); };              // the item's result is read
    const uint32_t done = bar1 + 8 * (NT * C::BARS_T);

    if (warp == 0) {
        if (lane < C::SLOTS) mbar_init(slot_full(lane), 1), mbar_init(slot_empty(lane), NT);
        if (lane < NT) {
            for (uint32_t b = 0; b < NS; ++b) mbar_init(s_full(lane, b), 1), mbar_init(p_full(lane, b), 4 * C::TPR), mbar_init(o_full(lane, b), 1);
            mbar_init(q_full(lane), 4 * C::TPR), mbar_init(o_free(lane), 4 * C::TPR);
        }
        if (lane == 0) {
            *abortp = 0, *made_finite = 0;
            mbar_init(done, NT);
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == C::MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(q4k::smem_u32(tmem_slot)), "r"(pf::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pf::tcgen05_fence_before();
    __syncthreads();
    pf::tcgen05_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    auto fail = [&](uint32_t role, uint32_t where) {
        *abortp = 1;
        *(volatile uint32_t *)p.status = (role << 24) | (where & 0xffffffu);
    };
    asm volatile("griddepcontrol.wait;" ::: "memory");

    L line;
    Cursor cur;
    uint32_t u = 0, u_end = 0;
    if (line.start(p, blockIdx.x, *reinterpret_cast<typename L::Shared *>(smem_raw + C::Q_BYTES), u, cur)) u_end = line.cut(blockIdx.x + 1);
    const uint32_t u_start = u;
    if (tid < 2) pending[tid].from = ~0u;
    fence_async_smem();  // the ring's next writer is the copy engine
    __syncthreads();
    // The item at the cursor, as every role sees it: n tiles of keys from k0 on, in `steps` steps.
    uint32_t n_units, n, steps, k0, row0, rows;
    auto item = [&] {
        n_units = line.units_to(cur, u, u_end);
        rows = cur.seq.news * p.group.d, row0 = cur.block * C::ROWS;
        uint32_t lo, hi;
        key_range(p, cur.seq, p.group.div(row0), p.group.div(min(row0 + C::ROWS, rows) - 1), lo, hi);
        k0 = (cur.first + cur.u0) * kTileKeys;
        const uint32_t k1 = min(k0 + n_units * kTileKeys, hi);
        n = k1 > k0 ? (k1 - k0 + kTileKeys - 1) / kTileKeys : 0;
        steps = k1 > k0 ? (k1 - k0 + C::SK - 1) / C::SK : 0;
    };
    // Tiles are loaded and used in the order K_0 .. K_(AHEAD-1), V_0, K_AHEAD, V_1, ...: where among them the item's V_j is.
    auto v_place = [&](uint32_t j) { return j + min(n, j + C::AHEAD); };
    uint32_t tiles = 0;  // of K and V, in front of the item

    if (warp == C::TMA_WARP) {
        // ------------------------------------------------ TMA ---
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
                    const uint32_t pg = (uint32_t)__ldcg(table + p.page.div(key));
                    if (pg < p.cache.num_pages) page = (int)pg, slot = (int)p.page.mod(key);
                }
            };
            constexpr uint32_t A = C::AHEAD;
            int pk[A + 1], sk[A + 1];  // pages of tiles j .. j + A
#pragma unroll
            for (uint32_t j = 0; j < A; ++j) {
                find(j, pk[j], sk[j]);
                if (j < n && ok) ok = load(&map_k, pk[j], sk[j]);
            }
            find(A, pk[A], sk[A]);
            for (uint32_t j = 0; j < n && ok; ++j) {
                int np, ns;
                find(j + A + 1, np, ns);
                ok = load(&map_v, pk[0], sk[0]);
                if (ok && j + A < n) ok = load(&map_k, pk[A], sk[A]);
#pragma unroll
                for (uint32_t i = 0; i < A; ++i) pk[i] = pk[i + 1], sk[i] = sk[i + 1];
                pk[A] = np, sk[A] = ns;
            }
            if (n_units != cur.units && lane == 0)
                pending[cur.u0 == 0] = Pending{cur, u - cur.u0}, expect_parts<DP, C::ROWS>(p, line, u - cur.u0);
            u += line.places(n_units);
            if (u < u_end) L::next(p, cur);
        }
        if (*abortp && lane == 0) {  // what is on its way must land before the block ends
            const long long t0 = clock64();
            for (uint32_t i = issued > C::SLOTS ? issued - C::SLOTS : 0; i < issued; ++i)
                while (!mbar_try(slot_full(i % C::SLOTS), (i / C::SLOTS) & 1u))
                    if (clock64() - t0 > 20000000ll) break;
        }
        __syncwarp();
    } else if (warp >= C::MMA_WARP) {
        // ------------------------------------------------ MMA ---
        constexpr uint32_t kBf16 = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // f32 += bf16 . bf16, M = 128
        const uint32_t idesc_qk = kBf16 | ((C::SK >> 3) << 17) | (tp.negate << 13);  // -A
        constexpr uint32_t idesc_pv = kBf16 | (1u << 16) | ((C::CPS * 64 >> 3) << 17);
        // A warp for each row tile: a wait takes the issuing warp 160 clocks even where nothing is left to wait for, as long as two
        // to four MMAs run. With two buffers of scores the softmax always has a next step, so it does not matter how the two interleave.
        const uint32_t t = warp - C::MMA_WARP;
        uint32_t used = 0, items = 0;  // steps, items of this row tile
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity, uint32_t role) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abortp));
            if (!ok && lane == 0) fail(role, tiles);
            return ok;
        };
        struct {  // the next slot in the order of use
            uint32_t at = 0, phase = 0;
        } head;
        uint32_t k_slot[C::SPT], v_slot[C::SPT];  // of the tile of K, of V in use
        auto take = [&](uint32_t (&slot)[C::SPT]) {
#pragma unroll
            for (uint32_t i = 0; i < C::SPT; ++i) {
                wait(slot_full(head.at), head.phase, 2);
                slot[i] = head.at;
                if (++head.at == C::SLOTS) head.at = 0, head.phase ^= 1u;
            }
            return ok;
        };
        while (u < u_end && ok) {
            item();
            auto scores = [&](uint32_t i) {  // of step i
                const uint32_t buf = (used + i) % NS, part = i % C::SPK;
                const uint32_t dst = tmem + C::S_COL + (t * NS + buf) * C::SK;
                const bool last = part + 1 == C::SPK || i + 1 == steps;  // of its tile of K
#pragma unroll
                for (uint32_t c = 0; c < C::CHUNKS; ++c) {
                    const uint32_t x = k_slot[c / C::CPS];
                    mma_ss4_elect(dst, pf::umma_desc_lo(q_smem + (t * C::CHUNKS + c) * C::CHUNK),
                                  pf::umma_desc_lo(ring + x * C::SLOT + (c % C::CPS) * C::CHUNK + part * (C::SK * 128)), idesc_qk, c);
                    if (c + 1 == C::CHUNKS) commit_elect(s_full(t, buf));
                    if ((c + 1) % C::CPS == 0 && last) commit_elect(slot_empty(x));
                }
            };
            if (row0 + t * 128 < rows) {
                if (n) wait(q_full(t), items & 1u, 3);
                for (uint32_t i = 0; i < NS && i < steps && ok; ++i) {
                    if (i % C::SPK == 0 && !take(k_slot)) break;
                    pf::tcgen05_fence_after();
                    scores(i);
                }
                for (uint32_t i = 0; i < steps && ok; ++i) {
                    const uint32_t part = i % C::SPK, x = used + i, buf = x % NS;
                    if (part == 0) take(v_slot);
                    if (i == 0 && items) wait(o_free(t), (items - 1) & 1u, 5);
                    if (!wait(p_full(t, buf), (x / NS) & 1u, 4)) break;
                    pf::tcgen05_fence_after();
                    const uint32_t a = tmem + C::S_COL + (t * NS + buf) * C::SK;
                    const bool last = part + 1 == C::SPK || i + 1 == steps;  // of its tile of V
#pragma unroll
                    for (uint32_t s = 0; s < C::SPT; ++s) {
#pragma unroll
                        for (uint32_t h = 0; h < C::TPR; ++h)  // weights of keys 64 h .. lie at columns 64 h ..
                            mma_ts4_elect(tmem + t * DP + s * C::CPS * 64, a + 64 * h,
                                          v_desc_lo(ring + v_slot[s] * C::SLOT, C::CHUNK) + (part * C::TPR + h) * 512, idesc_pv, i || h);
                        if (last) commit_elect(slot_empty(v_slot[s]));
                    }
                    if (i + NS >= steps) {
                        commit_elect(o_full(t, buf));
                    } else {
                        if ((i + NS) % C::SPK == 0 && !take(k_slot)) break;
                        pf::tcgen05_fence_after();
                        scores(i + NS);
                    }
                }
                if (n) used += steps, ++items;
            } else {  // no rows here: the slots go back as they come
                for (uint32_t i = 0; i < 2 * n && take(k_slot); ++i)
#pragma unroll
                    for (uint32_t s = 0; s < C::SPT; ++s)
                        if (lane == 0) mbar_arrive(slot_empty(k_slot[s]));
            }
            tiles += 2 * n;
            u += line.places(n_units);
            if (u < u_end) L::next(p, cur);
        }
        // Also after an abort: nothing may still read shared memory or TMEM when the block ends.
        commit_elect(done);
        const long long t0 = clock64();
        while (!mbar_try(done, 0u))
            if (clock64() - t0 > 4000000000ll) break;
        __syncwarp();
    } else {
        // ------------------------------------------------ softmax ---
        // Of TPR = 2 threads of a row each has keys 64 half .. of every step, and half of the result's columns.
        const uint32_t t = warp / (4 * C::TPR), half = (warp >> 2) & (C::TPR - 1), r = (warp & 3u) * 32 + lane;  // row tile, row
        const uint32_t lanes = (warp & 3u) << 21;                                           // this warp's quarter of the TMEM lanes
        const uint32_t o_tmem = tmem + lanes + t * DP, d = p.cache.head_dim;
        const uint32_t pair_bar = 1 + (warp & 3u);                                          // hardware barrier of the two warps of these rows
        volatile float *const x_base = reinterpret_cast<float *>(smem_raw + C::Q_BYTES + C::SLOTS * C::SLOT) + r;
        const float c2 = p.scale_log2;
        const uint64_t c2x2 = f32_pair(c2, c2);
        uint32_t used = 0, ends = 0;  // steps; bit b: the parity of o_full(b)'s phase
        bool ok = true;
        // A whole warp's wait: every lane waits, all go on or none.
        auto wait = [&](uint32_t bar, uint32_t parity, uint32_t role, uint32_t where) {
            ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abortp));
            if (!ok && lane == 0) fail(role, where);
            return ok;
        };
        // The two warps of a row meet. One that gives up has set the abort flag and then arrives once more, at the end of this role: the
        // other comes past the barrier with that, and sees the flag in front of its next one.
        auto meet = [&] {
            if (__any_sync(0xffffffffu, *abortp)) ok = false;
            if (C::TPR == 2 && ok) asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        };
        auto live = [&] { return u < u_end && row0 + t * 128 < rows; };  // the item at the cursor has rows here
        // Q of the item at the cursor. The scores of the one before have been read, so nothing reads its Q any more.
        auto load_q = [&] {
            if (!live() || n == 0) return;
            const uint32_t row = row0 + t * 128 + r;  // lane l knows where row l of the quarter's 32 lies; pieces of 16 bytes go by rows
            int64_t at = -1;
            if (row < rows) {
                uint32_t token, head;
                row_at(p, cur.seq, cur.kv_head, row, token, head);
                at = (int64_t)((size_t)token * p.q_stride + (size_t)head * d);
            }
#pragma unroll 4
            for (uint32_t i = lane + 32 * half; i < 32 * (DP / 8); i += 32 * C::TPR) {
                const uint32_t wr = i / (DP / 8), cc = i % (DP / 8), qr = (warp & 3u) * 32 + wr;
                const int64_t from = __shfl_sync(0xffffffffu, at, wr);
                const bool there = from >= 0 && cc * 8 < d;
                const uint32_t dst = q_smem + (t * C::CHUNKS + cc / 8) * C::CHUNK + qr * 128 + (((cc & 7u) ^ (qr & 7u)) << 4);
                cp_async16(dst, p.q + (there ? (size_t)from + cc * 8 : 0), there);
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
        // a's and b's halves of a 2 x 2 block of pieces between lanes `o` apart: afterwards a is piece (lane & o) of the lower lane, b of the upper.
        auto swap = [&](uint4 &a, uint4 &b, uint32_t o) {
            const bool upper = lane & o;
            uint32_t *x = &a.x, *y = &b.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? x[i] : y[i], o);
                if (upper) x[i] = got;
                else y[i] = got;
            }
        };
        if (u < u_end) item();
        load_q();
        q_ready();
        while (u < u_end) {
            const bool mine = live();
            const uint32_t row = row0 + t * 128 + r, n_steps = steps;
            float top = -INFINITY, off = 0.0f, sum = 0.0f;  // raw score that the weights refer to, as an exponent; sum of this thread's weights
            int64_t out_at = -1;  // where the row goes; -1: it is none
            if (mine) {
                uint32_t lo_r, hi_r;  // rows past the last see what that sees
                {
                    const uint32_t i = p.group.div(min(row, rows - 1));
                    key_range(p, cur.seq, i, i, lo_r, hi_r);
                }
                const uint32_t lo_all = __shfl_sync(0xffffffffu, lo_r, 31), hi_all = __shfl_sync(0xffffffffu, hi_r, 0);
                uint32_t lo_item, hi_item;  // what all rows of the item see: its row tiles read the same V
                {
                    uint32_t x;
                    const uint32_t i0 = p.group.div(row0), i1 = p.group.div(min(row0 + C::ROWS, rows) - 1);
                    key_range(p, cur.seq, i1, i1, lo_item, x), key_range(p, cur.seq, i0, i0, x, hi_item);
                }
                const int32_t *table = p.seqs.table + (size_t)cur.seq.index * p.seqs.max_pages;
                auto page_of = [&](uint32_t key) { return key < cur.seq.keys ? (uint32_t)__ldcg(table + p.page.div(key)) : 0u; };
                bool any_hole = false;  // a page of the item is not there: its tiles look at theirs
                for (uint32_t key = k0 + lane * tp.box; key < k0 + n * kTileKeys; key += 32 * tp.box) any_hole |= page_of(key) >= p.cache.num_pages;
                any_hole = __any_sync(0xffffffffu, any_hole);
                for (uint32_t i = 0; i < steps; ++i) {
                    const uint32_t x = used + i, buf = x % NS, key = k0 + i * C::SK + 64 * half;
                    const uint32_t s_tmem = tmem + lanes + C::S_COL + (t * NS + buf) * C::SK + 64 * half;  // scores, and the weights over them
                    const uint32_t holes = any_hole ? __ballot_sync(0xffffffffu, lane < 16 && page_of(key + 4 * lane) >= p.cache.num_pages) : 0u;
                    if (!wait(s_full(t, buf), (x / NS) & 1u, 6, i)) break;
                    pf::tcgen05_fence_after();
                    uint32_t s[64];
                    tmem_ld64(s_tmem, s);
                    if (holes || key < lo_all || key + 64 > hi_all) {
#pragma unroll
                        for (uint32_t y = 0; y < 64; ++y)
                            if (key + y < lo_r || key + y >= hi_r || ((holes >> (y / 4)) & 1u)) s[y] = 0xff800000u;
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (uint32_t y = 0; y < 64; y += 2) m4[y / 2 % 4] = max3(m4[y / 2 % 4], __uint_as_float(s[y]), __uint_as_float(s[y + 1]));
                    float m = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
                    if constexpr (C::TPR == 2) {
                        // The other thread's maximum. What it left here last it wrote for this row's last use of the buffer, whose product
                        // has waited for both threads since.
                        x_base[(buf * 2 + half) * 128] = m;
                        meet();
                        if (!ok) break;
                        m = fmaxf(m, x_base[(buf * 2 + (half ^ 1u)) * 128]);
                    }
                    const bool grow = (m - top) * c2 > 8.0f;  // never where both are -inf
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? exp2_fast((top - m) * c2) : 1.0f;
                        if (__any_sync(0xffffffffu, grow && top != -INFINITY)) {
                            // The product with V of the step before may still run: the next step's scores come behind it, or it has a
                            // barrier of its own.
                            const uint32_t other = (x + 1) % NS;
                            if (!(i + 1 < steps ? wait(s_full(t, other), ((x + 1) / NS) & 1u, 7, i) : wait(o_full(t, other), (ends >> other) & 1u, 12, i))) break;
                            pf::tcgen05_fence_after();
#pragma unroll 1
                            for (uint32_t y = half * (DP / C::TPR); y < (half + 1) * (DP / C::TPR); y += 16) {
                                uint32_t o[16];
                                tmem_ld16(o_tmem + y, o);
#pragma unroll
                                for (int z = 0; z < 16; ++z) o[z] = __float_as_uint(__uint_as_float(o[z]) * f);
                                tmem_store16(o_tmem + y, o);
                            }
                        }
                        if (grow) sum *= f, top = m, off = -top * c2;
                    }
                    const uint64_t offx2 = f32_pair(off, off);
                    uint64_t s2[2] = {0, 0};
                    uint32_t w[32];
#pragma unroll
                    for (uint32_t y = 0; y < 32; ++y) {
                        float a, b;
                        f32_unpair(fma2(f32_pair(__uint_as_float(s[2 * y]), __uint_as_float(s[2 * y + 1])), c2x2, offx2), a, b);
                        a = exp2_fast(a), b = exp2_fast(b);
                        s2[y & 1] = add2(s2[y & 1], f32_pair(a, b));
                        w[y] = bf16_pair(a, b);
                    }
                    tmem_store32(s_tmem, w);
                    const uint32_t step = k0 + i * C::SK;
                    if (step + C::SK > cur.seq.keys || some_unseen(cur.seq, step, C::SK, lo_item, hi_item)) {
                        // Two threads for a row of V. Slots behind the sequence: no values.
                        const uint32_t x = half * 128 + r, of = x % C::SK, j = i / C::SPK, v_row = i % C::SPK * C::SK + of;
                        const bool past = step + of >= cur.seq.keys, look = some_unseen(step + of, lo_item, hi_item);
                        if (__any_sync(0xffffffffu, past || look)) {
#pragma unroll 1
                            for (uint32_t y = 0; y < C::SPT; ++y) {
                                const uint32_t z = (tiles + v_place(j)) * C::SPT + y, at = ring + z % C::SLOTS * C::SLOT + v_row * 128;
                                if (!wait(slot_full(z % C::SLOTS), (z / C::SLOTS) & 1u, 8, j)) break;
#pragma unroll 1
                                for (uint32_t c = 0; c < C::CPS; ++c) {
                                    auto piece = [&](uint32_t k) { return at + c * C::CHUNK + (((x / C::SK * 4 + k) ^ (v_row & 7u)) << 4); };  // lanes on different banks
                                    if (past) {
#pragma unroll
                                        for (uint32_t k = 0; k < 4; ++k) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(piece(k)), "r"(0) : "memory");
                                    } else if (look && make_finite<4>(piece)) {
                                        *made_finite = 1;
                                    }
                                }
                            }
                            fence_async_smem();
                            __syncwarp();
                            if (!ok) break;
                        }
                    }
                    tmem_store_wait();
                    pf::tcgen05_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full(t, buf));
                    float a, b;
                    f32_unpair(add2(s2[0], s2[1]), a, b);
                    sum += a + b;
                }
                if (!ok) break;
                used += steps;
                if (row < rows) {
                    uint32_t token, head;
                    row_at(p, cur.seq, cur.kv_head, row, token, head);
                    out_at = (int64_t)(((size_t)token * p.n_heads + head) * d);
                }
            }
            const bool whole = n_units == cur.units;
            float *part = P::at(p.work, blockIdx.x, cur.u0 == 0);
            tiles += 2 * n;
            u += line.places(n_units);
            if (u < u_end) L::next(p, cur), item();
            load_q();  // of the next item, while the last product runs
            if (mine && n_steps) {
                const uint32_t last = (used - 1) % NS;
                if (!wait(o_full(t, last), (ends >> last) & 1u, 9, 0)) break;
                pf::tcgen05_fence_after();
                ends ^= n_steps > 1 ? 3u : 1u << last;
            }
            q_ready();
            if (!mine) continue;
            if constexpr (C::TPR == 2) {
                // The other thread's sum: it has read this row's last maximum, which the last product waited for; and this sum, in front
                // of the second barrier, before the next maximum comes.
                x_base[half * 128] = sum;
                meet();
                if (!ok) break;
                sum += x_base[(half ^ 1u) * 128];
                meet();
                if (!ok) break;
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            int64_t to[4];  // where the rows of this lane's quad go
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y) to[y] = __shfl_sync(0xffffffffu, out_at, (lane & ~3u) + y);
#pragma unroll 1
            for (uint32_t x = half * (DP / C::TPR); x < (half + 1) * (DP / C::TPR); x += 32) {
                if (x >= d) break;
                uint32_t o[32];
                if (n_steps) {
                    pf::tmem_ld32(o_tmem + x, o);
                } else {
#pragma unroll
                    for (int y = 0; y < 32; ++y) o[y] = 0;
                }
                if (whole) {
                    // A row per lane would touch 32 lines with each store: four lanes exchange their pieces of 16 bytes, so that
                    // each has one piece of four rows.
                    uint4 v[4];
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) {
                        v[y].x = bf16_pair(__uint_as_float(o[8 * y]) * inv, __uint_as_float(o[8 * y + 1]) * inv);
                        v[y].y = bf16_pair(__uint_as_float(o[8 * y + 2]) * inv, __uint_as_float(o[8 * y + 3]) * inv);
                        v[y].z = bf16_pair(__uint_as_float(o[8 * y + 4]) * inv, __uint_as_float(o[8 * y + 5]) * inv);
                        v[y].w = bf16_pair(__uint_as_float(o[8 * y + 6]) * inv, __uint_as_float(o[8 * y + 7]) * inv);
                    }
                    swap(v[0], v[1], 1), swap(v[2], v[3], 1), swap(v[0], v[2], 2), swap(v[1], v[3], 2);
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y)
                        if (to[y] >= 0 && x + 8 * (lane & 3u) < d) *reinterpret_cast<uint4 *>(p.out + to[y] + x + 8 * (lane & 3u)) = v[y];
                } else if (out_at >= 0) {
#pragma unroll
                    for (uint32_t y = 0; y < 32; y += 4)
                        *reinterpret_cast<uint4 *>(part + P::four(t * 128 + r, (x + y) / 4)) = make_uint4(o[y], o[y + 1], o[y + 2], o[y + 3]);
                }
                __syncwarp();
            }
            if (!whole && out_at >= 0 && half == 0) part[P::TOP + t * 128 + r] = top == -INFINITY ? top : top * c2, part[P::SUM + t * 128 + r] = sum;
            if (n_steps) {
                pf::tcgen05_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_free(t));
            }
        }
        __syncwarp();
        if (C::TPR == 2 && !ok) asm volatile("bar.arrive %0, 64;" ::"r"(pair_bar) : "memory");
    }
    pf::tcgen05_fence_before();
    __syncthreads();
    if (warp == C::MMA_WARP) {
        pf::tcgen05_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(pf::kTmemCols) : "memory");
    }
    if (*abortp || u_start >= u_end) return;
    if (*made_finite) {
        add_not_finite<DP, C::ROWS, kTileKeys, L>(p, *reinterpret_cast<typename L::Shared *>(smem_raw + C::Q_BYTES), C::THREADS);
        __syncthreads();
    }
    const bool has[2] = {pending[0].from != ~0u, pending[1].from != ~0u};
    finish_parts<DP, C::ROWS>(p, line, pending, has, C::THREADS, reinterpret_cast<volatile uint32_t *>(smem_raw + C::SMEM - 16),
                         reinterpret_cast<float *>(smem_raw), (C::Q_BYTES + C::SLOTS * C::SLOT) / 4);
}

}  // namespace attn
}  // namespace tessl
