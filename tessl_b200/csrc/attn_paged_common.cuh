// What the attention kernels over a paged cache share: the launch parameters, the ranges of keys that rows see, and the division
// of a call's work among the blocks of a launch.
//
// The rows of one sequence and key head are its new tokens times the `group` query heads that read that key head, token by
// token: they all multiply the same keys. A block of rows of them is an item, its keys come in units, and all units of the
// call, item after item, are one line that is cut into equal parts, one per block of the launch: whatever the lengths of the
// sequences, every block reads the same number of keys. The lengths are on the device, so the blocks work the cuts out
// themselves. A block that has an item to itself writes its rows; the parts of an item that a cut divides go to the workspace,
// two at most per block (the end of one item, the start of another). A block counts its parts in when it is done: the last one of an
// item to come adds the parts up, in an order that their number alone decides: the same sums on every run. (A second launch took 9 us
// of the 18 of a token over 777 keys, and 21 of 74 of ragged chunks.)
#pragma once
#include "paged_common.cuh"
#include "q4_gemv_tma.cuh"

namespace tessl {
namespace attn {

using paged::bf16_pair;

/// Division by a number that is the same for a whole launch, exact for every 32-bit dividend: the multiplication by a rounded-up
/// reciprocal of Granlund and Montgomery. (The compiler's division is some thirty instructions, and what a block does once it runs from
/// a cold instruction cache.)
struct Divisor {
    uint32_t d, m, s1, s2;
    static Divisor of(uint32_t d)  // d >= 1
    {
        uint32_t l = 0;
        while (l < 32 && (uint64_t(1) << l) < d) ++l;
        return Divisor{d, (uint32_t)(((uint64_t(1) << 32) * ((uint64_t(1) << l) - d)) / d + 1), l < 1 ? l : 1, l > 0 ? l - 1 : 0};
    }
    __device__ __forceinline__ uint32_t div(uint32_t x) const
    {
        const uint32_t t = __umulhi(m, x);
        return (t + ((x - t) >> s1)) >> s2;
    }
    __device__ __forceinline__ uint32_t mod(uint32_t x) const { return x - div(x) * d; }
};

struct Params {
    const uint16_t *q;
    uint16_t *out;
    float *work;
    paged::Cache cache;
    paged::Seqs seqs;
    uint32_t q_stride, n_heads;
    Divisor group;  // query heads of a key head
    Divisor page;   // tokens
    float scale_log2;  // scale * log2 e
    uint32_t causal, window;
    uint32_t parts;      // blocks that the line of units may be cut for
    uint64_t mark;       // of this call's items: 48 bits
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

/// The keys of the item of rows block * ROWS ..: its first unit and how many units it has, one at least (rows that see nothing are
/// written too).
template <uint32_t ROWS, uint32_t UNIT>
__device__ __forceinline__ void block_units(const Params &p, const Seq &q, uint32_t block, uint32_t &first, uint32_t &units)
{
    const uint32_t rows = q.news * p.group.d, r0 = block * ROWS;
    uint32_t lo, hi;
    key_range(p, q, p.group.div(r0), p.group.div(min(r0 + ROWS, rows) - 1), lo, hi);
    first = lo / UNIT;
    units = max(1u, (hi + UNIT - 1) / UNIT - first);
}
template <uint32_t ROWS>
__device__ __forceinline__ uint32_t blocks_of(const Params &p, const Seq &q)
{
    return (q.news * p.group.d + ROWS - 1) / ROWS;
}

/// An item, and where in it a part begins.
struct Cursor {
    Seq seq;
    uint32_t kv_head, blocks, block, first, units, u0;
};
/// An item of which a block has a part, and where the item begins on the line.
struct Pending {
    Cursor c;
    uint32_t from;
};

/// The line of the call's work (key heads, in each the sequences, in each the blocks of rows) and how it is cut: its units, or, where
/// cutting items would cost more than it gives, whole items. EXTRA: what an item's second part costs, in units.
template <uint32_t ROWS, uint32_t UNIT, uint32_t THREADS, uint32_t EXTRA>
struct Line {
    /// Of some sequences, for one key head. The host has made sure that the units of a call whose offsets ascend are below 2^32.
    struct Count {
        uint32_t units, blocks, most;  // most: units of one block; ~0: offsets that descend
        __device__ __forceinline__ void add(uint32_t u, uint32_t b, uint32_t m) { units += u, blocks += b, most = max(most, m); }
    };
    struct Shared {
        Count warp_sum[THREADS / 32], cost[THREADS];
        uint32_t many[THREADS], n_many, found_at;
        Seq found;
    };
    uint32_t per_head, parts;
    uint32_t span, cuts;    // every `span` places are cut for themselves, into this many parts:
    uint32_t each, longer;  // the first `longer` of them have each + 1 places, the others `each`
    bool whole;             // items are not cut: the line counts items

    __device__ __forceinline__ uint32_t cut(uint32_t c) const
    {
        const uint32_t i = cuts == parts ? (c >= parts) : c / cuts, k = c - i * cuts;
        return i * span + each * k + min(k, longer);
    }
    /// The part that holds place u.
    __device__ __forceinline__ uint32_t part_of(uint32_t u) const
    {
        const uint32_t i = cuts == parts ? 0 : u / span, v = u - i * span, edge = (each + 1) * longer;
        return i * cuts + (v < edge ? v / (each + 1) : longer + (v - edge) / each);
    }
    /// Units of the item at the cursor that lie between places u and u_end, and how far they reach.
    __device__ __forceinline__ uint32_t units_to(const Cursor &c, uint32_t u, uint32_t u_end) const
    {
        return whole ? c.units : min(c.units - c.u0, u_end - u);
    }
    __device__ __forceinline__ uint32_t places(uint32_t units) const { return whole ? 1 : units; }

    /// Every `step`-th block of a sequence from b0 on.
    static __device__ __forceinline__ Count count(const Params &p, const Seq &q, uint32_t blocks, uint32_t b0, uint32_t step)
    {
        Count c{0, 0, 0};
        for (uint32_t b = b0; b < blocks; b += step) {
            uint32_t first, units;
            block_units<ROWS, UNIT>(p, q, b, first, units);
            c.add(units, 1, units);
        }
        return c;
    }
    static __device__ __forceinline__ Count warp_total(Count c)
    {
#pragma unroll
        for (uint32_t o = 16; o > 0; o /= 2)
            c.add(__shfl_xor_sync(0xffffffffu, c.units, o), __shfl_xor_sync(0xffffffffu, c.blocks, o), __shfl_xor_sync(0xffffffffu, c.most, o));
        return c;
    }

    /// Counts this thread's sequence s0 + threadIdx.x: what lies in front of it among those of the block, itself (`mine`), all (`sum`).
    /// Sequences of many blocks of rows are counted by a warp each.
    static __device__ Count scan(const Params &p, uint32_t s0, Shared &sh, Seq &q, Count &mine, Count &sum)
    {
        const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = s0 + tid;
        __syncthreads();  // sh may still be read
        if (tid == 0) sh.n_many = 0;
        __syncthreads();
        mine = Count{0, 0, 0};
        bool many = false;
        if (s < p.seqs.num_seqs) {
            q = seq_at(p, s);
            const uint32_t blocks = blocks_of<ROWS>(p, q);
            many = blocks > 2;
            if (blocks == 0 && paged::start_of(p.seqs, s + 1) < q.row0) mine.most = ~0u;
            if (many) sh.many[atomicAdd(&sh.n_many, 1u)] = tid;
            else if (blocks) mine = count(p, q, blocks, 0, 1);
        }
        __syncthreads();
        for (uint32_t i = warp; i < sh.n_many; i += THREADS / 32) {
            const Seq r = seq_at(p, s0 + sh.many[i]);
            const Count c = warp_total(count(p, r, blocks_of<ROWS>(p, r), lane, 32));
            if (lane == 0) sh.cost[sh.many[i]] = c;
        }
        if (sh.n_many) __syncthreads();
        if (many) mine = sh.cost[tid];
        Count run = mine;
#pragma unroll
        for (uint32_t o = 1; o < 32; o *= 2) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, run.units, o), b = __shfl_up_sync(0xffffffffu, run.blocks, o), m = __shfl_up_sync(0xffffffffu, run.most, o);
            if (lane >= o) run.add(t, b, m);
        }
        if (lane == 31) sh.warp_sum[warp] = run;
        __syncthreads();
        Count before{0, 0, 0};
        sum = before;
#pragma unroll
        for (uint32_t w = 0; w < THREADS / 32; ++w) {
            const Count &t = sh.warp_sum[w];
            if (w < warp) before.add(t.units, t.blocks, 0);
            sum.add(t.units, t.blocks, t.most);
        }
        before.add(run.units - mine.units, run.blocks - mine.blocks, 0);
        return before;
    }

    /// The whole block calls this, and has one of: no part (false), or in `from` its place in the line and the item there. The
    /// sequences are gone over twice where a block's threads do not hold them all.
    __device__ bool start(const Params &p, uint32_t part, Shared &sh, uint32_t &from, Cursor &c)
    {
        const uint32_t n = p.seqs.num_seqs, lane = threadIdx.x & 31;
        Count mine, sum, all, at;
        uint32_t found_at = 0;
        Seq q;
        if (n == 1) {  // every warp for itself
            q = seq_at(p, 0);
            const uint32_t blocks = blocks_of<ROWS>(p, q);
            all = blocks == 1 ? count(p, q, 1, 0, 1) : warp_total(count(p, q, blocks, lane, 32));
        } else {
            at = scan(p, 0, sh, q, mine, sum);
            all = sum;
            for (uint32_t s0 = THREADS; s0 < n; s0 += THREADS) {
                Count m, t;
                Seq other;
                scan(p, s0, sh, other, m, t);
                all.add(t.units, t.blocks, t.most);
            }
        }
        if (all.most == ~0u) return false;
        // The longest part: units cut evenly and an item's second part, or as many of the largest items as a part has items.
        const uint32_t items = all.blocks * p.cache.n_kv_heads, units = all.units * p.cache.n_kv_heads;
        whole = (items + p.parts - 1) / p.parts * (uint64_t)all.most <= units / p.parts + EXTRA;
        const uint32_t total = whole ? items : units;
        per_head = whole ? all.blocks : all.units;
        span = total, cuts = min(p.parts, total);
        // A few items of the same length: no block has parts of two, which cost a token over 3000 keys 20 us instead of 14.5.
        if (!whole && all.most * all.blocks == all.units && items <= p.parts) {
            const uint32_t k = min(p.parts / items, all.most);
            if ((all.most + k - 1) / k <= units / p.parts + EXTRA / 2) span = all.most, cuts = k;
        }
        parts = span == total ? cuts : items * cuts;
        if (part >= parts) return false;
        each = span / cuts, longer = span - each * cuts;
        from = cut(part);
        c.kv_head = from / per_head;
        const uint32_t in_head = from - c.kv_head * per_head;
        if (n > 1) {
            uint32_t before = 0;
            for (uint32_t s0 = 0; s0 < n; s0 += THREADS) {
                if (n > THREADS) at = scan(p, s0, sh, q, mine, sum);
                const uint32_t place = before + (whole ? at.blocks : at.units);
                if (place <= in_head && in_head < place + (whole ? mine.blocks : mine.units)) sh.found = q, sh.found_at = place;
                before += whole ? sum.blocks : sum.units;
                if (in_head < before) break;
            }
            __syncthreads();
            q = sh.found, found_at = sh.found_at;
        }
        c.seq = q;
        c.blocks = blocks_of<ROWS>(p, c.seq);
        uint32_t rest = in_head - found_at;
        if (whole || c.blocks == 1) {
            c.block = whole ? rest : 0, c.u0 = whole ? 0 : rest;
            block_units<ROWS, UNIT>(p, c.seq, c.block, c.first, c.units);
            return true;
        }
        for (uint32_t b0 = 0;; b0 += 32) {  // every warp for itself
            uint32_t first = 0, units = 0;
            if (b0 + lane < c.blocks) block_units<ROWS, UNIT>(p, c.seq, b0 + lane, first, units);
            uint32_t run = units;
#pragma unroll
            for (uint32_t o = 1; o < 32; o *= 2) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += t;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, run > rest);
            if (past || b0 + 32 >= c.blocks) {
                const uint32_t l = past ? __ffs(past) - 1 : 0;
                c.block = b0 + l;
                c.first = __shfl_sync(0xffffffffu, first, l), c.units = __shfl_sync(0xffffffffu, units, l);
                c.u0 = rest - (__shfl_sync(0xffffffffu, run, l) - c.units);
                break;
            }
            rest -= __shfl_sync(0xffffffffu, run, 31);
        }
        return true;
    }

    /// The item behind this one. Only where the line goes on.
    static __device__ void next(const Params &p, Cursor &c)
    {
        c.u0 = 0;
        if (++c.block >= c.blocks) {
            c.block = 0;
            do {
                uint32_t s = c.seq.index + 1;
                if (s >= p.seqs.num_seqs) s = 0, ++c.kv_head;
                c.seq = seq_at(p, s);
                c.blocks = blocks_of<ROWS>(p, c.seq);
            } while (c.blocks == 0);
        }
        block_units<ROWS, UNIT>(p, c.seq, c.block, c.first, c.units);
    }
};

/// A part of an item in the workspace: ROWS rows of DP unnormalised sums, four columns of all rows after four of all rows, then
/// the rows' maxima (in powers of two) and sums. Behind the parts a counter for each block: of the item whose start it has.
template <uint32_t ROWS, uint32_t DP>
struct Part {
    static constexpr uint32_t FLOATS = ROWS * DP + 2 * ROWS, TOP = ROWS * DP, SUM = TOP + ROWS;
    static constexpr uint64_t bytes(uint64_t parts) { return parts * (2 * FLOATS * sizeof(float) + sizeof(uint64_t)); }
    /// `head`: the start of an item, else its middle or end.
    static __device__ __forceinline__ float *at(float *work, uint32_t part, bool head) { return work + ((size_t)part * 2 + head) * FLOATS; }
    static __device__ __forceinline__ uint32_t four(uint32_t row, uint32_t col4) { return (col4 * ROWS + row) * 4; }
    static __device__ __forceinline__ unsigned long long *counter(const Params &p, uint32_t part)
    {
        return reinterpret_cast<unsigned long long *>(p.work + (size_t)p.parts * 2 * FLOATS) + part;
    }
};

__device__ __forceinline__ float exp2_fast(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

/// Row r of a sequence and key head: its row of q and out, in heads.
__device__ __forceinline__ void row_at(const Params &p, const Seq &q, uint32_t kv_head, uint32_t r, uint32_t &token, uint32_t &head)
{
    token = p.group.div(r);
    head = kv_head * p.group.d + (r - token * p.group.d);
    token += q.row0;
}

// Values that are not finite, of keys that some rows of an item see and others do not: a weight of 0 times such a value is NaN, so the
// kernels make zeros of them in shared memory and note that they did. A block that has done so adds them, at its end, to the rows that see
// them. All rows of the item see [lo_all, hi_all).

__device__ __forceinline__ bool some_unseen(uint32_t key, uint32_t lo_all, uint32_t hi_all) { return key < lo_all || key >= hi_all; }
/// The same of any of the sequence's keys in [key, key + n).
__device__ __forceinline__ bool some_unseen(const Seq &q, uint32_t key, uint32_t n, uint32_t lo_all, uint32_t hi_all)
{
    return key < lo_all || min(key + n, q.keys) > hi_all;
}
/// N times eight bf16 values at shared-memory addresses at(0) .., those that are not finite made zero: whether there were any.
template <int N, typename F>
__device__ __forceinline__ bool make_finite(F at)
{
    uint32_t w[N][4], bad = 0;
#pragma unroll
    for (int k = 0; k < N; ++k)
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[k][0]), "=r"(w[k][1]), "=r"(w[k][2]), "=r"(w[k][3]) : "r"(at(k)) : "memory");
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= (w[k][i] & 0x7f807f80u) + 0x00800080u;  // an exponent of ones carries into the sign's place
    if (!(bad & 0x80008000u)) return false;
#pragma unroll
    for (int k = 0; k < N; ++k) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((w[k][i] & 0x7f80u) == 0x7f80u) w[k][i] &= 0xffff0000u;
            if ((w[k][i] & 0x7f800000u) == 0x7f800000u) w[k][i] &= 0xffffu;
        }
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at(k)), "r"(w[k][0]), "r"(w[k][1]), "r"(w[k][2]), "r"(w[k][3]) : "memory");
    }
    return true;
}
/// The block's items once more. All threads, behind a barrier. (Not inlined, the call's conventions cost a kernel that never came here
/// 12 us of 119.)
template <uint32_t DP, uint32_t ROWS, uint32_t UNIT, typename L>
__device__ __forceinline__ void add_not_finite(const Params &p, typename L::Shared &sh, uint32_t threads)
{
    using P = Part<ROWS, DP>;
    L line;
    Cursor cur;
    uint32_t u;
    if (!line.start(p, blockIdx.x, sh, u, cur)) return;
    const uint32_t u_end = line.cut(blockIdx.x + 1), d = p.cache.head_dim;
    while (u < u_end) {
        const Seq &q = cur.seq;
        const uint32_t n_units = line.units_to(cur, u, u_end), row0 = cur.block * ROWS, end = min(row0 + ROWS, q.news * p.group.d);
        const uint32_t i0 = p.group.div(row0), i1 = p.group.div(end - 1);
        uint32_t lo, hi, lo_all, hi_all, t;
        key_range(p, q, i0, i1, lo, hi), key_range(p, q, i1, i1, lo_all, t), key_range(p, q, i0, i0, t, hi_all);
        const uint32_t k0 = (cur.first + cur.u0) * UNIT, k1 = min(k0 + n_units * UNIT, hi);
        float *part = P::at(p.work, blockIdx.x, cur.u0 == 0);
        for (uint32_t key = max(k0, lo); key < k1; ++key) {
            if (!some_unseen(key, lo_all, hi_all)) {
                key = min(hi_all, k1) - 1;
                continue;
            }
            const uint32_t page = (uint32_t)__ldcg(p.seqs.table + (size_t)q.index * p.seqs.max_pages + p.page.div(key));
            if (page >= p.cache.num_pages) continue;
            const uint16_t *v = p.cache.v + page * p.cache.page_stride + (uint64_t)p.page.mod(key) * p.cache.token_stride +
                                (uint64_t)cur.kv_head * p.cache.head_stride;
            for (uint32_t c = threadIdx.x; c < d; c += threads) {
                const uint32_t bits = __ldcg(v + c);
                if ((bits & 0x7f80u) != 0x7f80u) continue;
                const float x = __uint_as_float(bits << 16);
                for (uint32_t r = row0; r < end; ++r) {
                    uint32_t token = p.group.div(r), head, lo_r, hi_r;
                    key_range(p, q, token, token, lo_r, hi_r);
                    if (key < lo_r || key >= hi_r) continue;
                    row_at(p, q, cur.kv_head, r, token, head);
                    if (n_units == cur.units) {
                        uint16_t *at = p.out + ((size_t)token * p.n_heads + head) * d + c;
                        *at = (uint16_t)bf16_pair(__uint_as_float((uint32_t)*at << 16) + x, 0.0f);
                    } else {
                        part[P::four(r - row0, c / 4) + c % 4] += x;
                    }
                }
            }
        }
        u += line.places(n_units);
        if (u < u_end) L::next(p, cur);
    }
}

/// Before a barrier in front of finish_parts, by one thread, for each item (where it begins on the line) of which the block has a part: a counter that does not hold a number of
/// this call's own and a count holds what another call or nobody has put there, and is given the number and a count of 0 by the first block
/// to see that. Whoever has added up puts the count back to 0, for a replay of this call has the same number.
template <uint32_t DP, uint32_t ROWS, typename L>
__device__ __forceinline__ void expect_parts(const Params &p, const L &l, uint32_t from)
{
    unsigned long long *const at = Part<ROWS, DP>::counter(p, l.part_of(from));
    const unsigned long long seen = __ldcg(at);
    if (seen >> 16 != p.mark) atomicCAS(at, seen, p.mark << 16);
}

/// The end of a block: its parts, one of the item that it began in the middle of (pending[0]) and one of the item whose start it has
/// (pending[1]), are counted in and, where it is the last of an item's blocks to come, added up. All threads call this behind a
/// barrier that follows the last store to the workspace; `came`: two words of shared memory, `shared`: `room`
/// words that nobody uses any longer, 16 for each thread and many times the two of every part's row.
///
/// The counters need no preparation: each of an item's blocks has called expect_parts before. (Counting in by compare and swap alone,
/// which needs no call before, took the twenty blocks of an item up to 7 us.)
template <uint32_t DP, uint32_t ROWS, typename L>
__device__ void finish_parts(const Params &p, const L &l, const Pending *pending, const bool (&has)[2], uint32_t threads,
                             volatile uint32_t *came, float *shared, uint32_t room)
{
    using P = Part<ROWS, DP>;
    if (!has[0] && !has[1]) return;
    const uint32_t tid = threadIdx.x, d = p.cache.head_dim;
    if (tid == 0) {
        // Releases the block's parts, behind the barrier that all have passed, and acquires those of the blocks before.
        unsigned long long old[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (has[i])
                asm volatile("atom.acq_rel.gpu.global.add.u64 %0, [%1], 1;" : "=l"(old[i]) : "l"(P::counter(p, l.part_of(pending[i].from))) : "memory");
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (has[i]) came[i] = (uint32_t)(old[i] & 0xffffu) + 1;
    }
    __syncthreads();
    for (uint32_t i = 0; i < 2; ++i) {
        if (!has[i]) continue;
        const Pending &w = pending[i];
        const uint32_t first = l.part_of(w.from), last = l.part_of(w.from + w.c.units - 1);
        if (came[i] != last - first + 1) continue;
        const Seq &q = w.c.seq;
        const uint32_t all_rows = min(q.news * p.group.d - w.c.block * ROWS, ROWS), n = last - first + 1;
        const uint32_t step = min(all_rows, (room - 16 * threads - 4) / (2 * n));
        for (uint32_t r0 = 0; r0 < all_rows; r0 += step) {
            const uint32_t rows = min(step, all_rows - r0);
            // Maxima and sums of the parts' rows, all loads at once; then what each part counts for, of each row. [part][row]
            float *const factor = shared, *const sum = shared + n * rows;
            for (uint32_t z = tid; z < n * rows; z += threads) {
                const uint32_t k = z / rows;
                const float *a = P::at(p.work, first + k, k == 0) + r0 + (z - k * rows);
                factor[z] = __ldcg(a + P::TOP), sum[z] = __ldcg(a + P::SUM);
            }
            __syncthreads();
            // `lanes` of a warp for each row, a part each.
            uint32_t lanes = 1;
            while (lanes < n && lanes < 32) lanes *= 2;
            for (uint32_t z = tid; z < (rows * lanes + 31) / 32 * 32; z += threads) {
                const uint32_t r = min(z / lanes, rows - 1), k0 = z & (lanes - 1);
                const bool mine = z < rows * lanes;
                float m = -INFINITY, all = 0.0f;
                for (uint32_t k = k0; k < n; k += lanes) m = fmaxf(m, factor[k * rows + r]);
                for (uint32_t x = 1; x < lanes; x *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
                const float ref = m == -INFINITY ? 0.0f : m;
                for (uint32_t k = k0; k < n; k += lanes) all += sum[k * rows + r] * exp2_fast(factor[k * rows + r] - ref);
                for (uint32_t x = 1; x < lanes; x *= 2) all += __shfl_xor_sync(0xffffffffu, all, x);
                const float inv = all == 0.0f ? 0.0f : 1.0f / all;
                if (mine)
                    for (uint32_t k = k0; k < n; k += lanes) factor[k * rows + r] = exp2_fast(factor[k * rows + r] - ref) * inv;
                __syncwarp();
            }
            __syncthreads();
            // A thread has four fours of columns of a row (32 bytes of the result, a sector) in every `groups`-th part; the groups' sums
            // meet in shared memory.
            const uint32_t wide = (d + 15) / 16, each = rows * wide, groups = max(1u, min(n, threads / each));
            float4 *const met = reinterpret_cast<float4 *>(shared + (2 * n * rows + 3) / 4 * 4);
            for (uint32_t z = tid; z < each * groups; z += threads) {
                const uint32_t g = z / each, y0 = z - g * each, r = y0 % rows, x0 = y0 / rows * 4;
                float4 o[4];
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y) o[y] = make_float4(0, 0, 0, 0);
#pragma unroll 4
                for (uint32_t k = g; k < n; k += groups) {
                    const float *a = P::at(p.work, first + k, k == 0);
                    const float f = factor[k * rows + r];
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) {
                        if ((x0 + y) * 4 >= d) continue;
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(a + P::four(r0 + r, x0 + y)));
                        o[y].x = fmaf(v.x, f, o[y].x), o[y].y = fmaf(v.y, f, o[y].y), o[y].z = fmaf(v.z, f, o[y].z), o[y].w = fmaf(v.w, f, o[y].w);
                    }
                }
                if (groups > 1) {
#pragma unroll
                    for (uint32_t y = 0; y < 4; ++y) met[y * each * groups + z] = o[y];
                    continue;
                }
                uint32_t token, head;
                row_at(p, q, w.c.kv_head, w.c.block * ROWS + r0 + r, token, head);
                uint16_t *out = p.out + ((size_t)token * p.n_heads + head) * d;
#pragma unroll
                for (uint32_t y = 0; y < 4; ++y)
                    if ((x0 + y) * 4 < d)
                        *reinterpret_cast<uint2 *>(out + (x0 + y) * 4) = make_uint2(bf16_pair(o[y].x, o[y].y), bf16_pair(o[y].z, o[y].w));
            }
            if (groups > 1) {
                __syncthreads();
                for (uint32_t z = tid; z < each * 4; z += threads) {
                    const uint32_t y = z / each, y0 = z - y * each, r = y0 % rows, x = y0 / rows * 4 + y;
                    if (x * 4 >= d) continue;
                    float4 o = make_float4(0, 0, 0, 0);
                    for (uint32_t g = 0; g < groups; ++g) {
                        const float4 v = met[(y * groups + g) * each + y0];
                        o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
                    }
                    uint32_t token, head;
                    row_at(p, q, w.c.kv_head, w.c.block * ROWS + r0 + r, token, head);
                    *reinterpret_cast<uint2 *>(p.out + ((size_t)token * p.n_heads + head) * d + x * 4) = make_uint2(bf16_pair(o.x, o.y), bf16_pair(o.z, o.w));
                }
            }
            __syncthreads();  // shared memory is read
        }
        if (tid == 0) *P::counter(p, first) = p.mark << 16;
    }
}

}  // namespace attn
}  // namespace tessl
