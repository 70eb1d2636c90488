// Rotary positions, and the append of new keys and values to a paged cache with the rotation (and the heads' norm) on the way.
//
// Pair i of a head turns by position * w_i radians. The angle is kept in turns as a 64-bit fraction: steps[i] =
// round(2^64 w_i / 2 pi), and position * steps[i] modulo 2^64 is the angle modulo one turn with an error below position * 2^-65 turns,
// for any 32-bit position. (position * w_i in f32 is off by 0.06 radians at position 10^6.) Its high 32 bits, 2^-32 turns or 1.5e-9
// radians, are enough for f32: two of them are the quadrant, the rest the sine and cosine of an eighth of a turn at most.
//
// One kernel for both operators: a warp has a token, or a share of its heads where tokens are few. A lane holds two runs of four columns
// of a head, which are the two halves of four pairs or four whole pairs, so a rotation needs no exchange, the norm one butterfly, and
// the lane's cosines and sines serve all heads of the token. The heads' values are on their way while the position is
// found (offset -> length -> page id, three round trips to L2). Bound by memory from some thousand tokens on, by those
// round trips below. (With a block per token, whose threads shared the angles through shared memory and a barrier, 8192 x 32 heads of
// 128 took 46 us.)
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_common.cuh"

namespace tessl {
namespace {

using paged::bf16_pair;

constexpr uint32_t kThreads = 32;  // a warp: blocks of four ended later, 8192 tokens x 32 heads of 128 in 31.1 us instead of 26.9
constexpr uint32_t kMaxPairs = 128;  // of a head of 256

struct HeadsParams {
    const void *src[3];  // q, k, v (or x alone)
    uint32_t src_stride[3];
    uint32_t heads[2];   // of q, of k and v each
    void *out;
    uint32_t out_stride;
    paged::Cache cache;
    paged::Seqs seqs;
    const int32_t *positions;
    const uint64_t *steps;
    const float *norm_w[2];  // of q, of k; null: no norm
    float eps, factor;
    uint32_t tokens, dim, rot, interleaved;
    uint32_t lanes;   // per head, a power of two
    uint32_t splits;  // warps that share the heads of a token
};

/// A run of VEC columns as it lies in memory: 16 bytes, or 8, or one value.
template <bool IN16, int VEC>
struct Run {
    uint32_t w[VEC == 1 ? 1 : IN16 ? VEC / 2 : VEC];
    __device__ __forceinline__ void load(const void *src, size_t at)
    {
        if constexpr (VEC == 4 && IN16) {
            const uint2 v = dev::ld_after_wait8(static_cast<const uint16_t *>(src) + at);
            w[0] = v.x, w[1] = v.y;
        } else if constexpr (VEC > 1) {
            const uint4 v = IN16 ? dev::ld_after_wait16(static_cast<const uint16_t *>(src) + at) : dev::ld_after_wait16(static_cast<const float *>(src) + at);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (IN16) {
            w[0] = (uint32_t)__ldcg(static_cast<const unsigned short *>(src) + at) << 16;
        } else {
            w[0] = __float_as_uint(__ldcg(static_cast<const float *>(src) + at));
        }
    }
    __device__ __forceinline__ void get(float (&v)[VEC]) const
    {
        if constexpr (VEC > 1 && IN16) {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) v[2 * i] = dev::bf16_lo(w[i]), v[2 * i + 1] = dev::bf16_hi(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(w[i]);
        }
    }
};

template <bool OUT16, int VEC>
__device__ __forceinline__ void store_run(void *dst, size_t at, const float (&v)[VEC])
{
    if constexpr (VEC == 8 && OUT16) {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(dst) + at) =
            make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
    } else if constexpr (VEC == 4 && OUT16) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(dst) + at) = make_uint2(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]));
    } else if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4)
            *reinterpret_cast<float4 *>(static_cast<float *>(dst) + at + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else if constexpr (OUT16) {
        static_cast<uint16_t *>(dst)[at] = (uint16_t)bf16_pair(v[0], 0.0f);
    } else {
        static_cast<float *>(dst)[at] = v[0];
    }
}

/// factor * (cos, sin) of 2 pi angle / 2^32. Polynomials with the least relative error for |x| <= 1/4 (Remez, the leading coefficients
/// held at their f32 values while the others are fitted): sin(pi x) = pi x + (d x + x^3 P(x^2)) to 3.4e-9, cos(pi x) = Q(x^2) to 6.4e-10 with the
/// coefficients as they stand here. d is what f32 leaves out of pi. With the rounding in f32 both are within
/// 2.5 * 2^-24 of themselves (1.82 and 1.59 over 5 million angles); pi in one f32 took the sine to 2.9. (With d in P's place, the compiler
/// ordered the loads of the kernel below otherwise: 8192 tokens x 32 heads of 128 in 29.4 us instead of 25.9.)
__device__ __forceinline__ float2 turn_of(uint32_t angle, float factor)
{
    const uint32_t quadrant = (angle + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(angle - (quadrant << 30)) * 0x1p-31f, t = x * x;
    const float odd = x * t * fmaf(fmaf(-0.5890811086f, t, 2.5497686863f), t, -5.1677079201f);
    const float s = fmaf(x, 3.1415927410f, fmaf(x, -9.571968462e-8f, odd));
    const float c = fmaf(fmaf(fmaf(fmaf(0.2289538831f, t, -1.3347475529f), t, 4.0586962700f), t, -4.9348020554f), t, 1.0f);
    const float sf = quadrant & 2u ? -factor : factor, cf = (quadrant + 1) & 2u ? -factor : factor;
    return quadrant & 1u ? make_float2(cf * s, sf * c) : make_float2(cf * c, sf * s);
}

/// Through L1: all warps read the same few lines (from L2, 8192 tokens x 32 heads of 128 took 31 us instead of 27).
__device__ __forceinline__ uint64_t step_of(const uint64_t *p)
{
    uint64_t v;
    asm volatile("ld.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}

/// VEC = 8 (bf16 in) or 4: rot and the rest of a head multiples of 2 VEC and everything aligned for whole runs. VEC = 1: anything else,
/// 32 lanes per head. PAGED: rows find their sequence, positions come from the lengths, k and v go to the cache; else positions are given.
/// NORM: heads of q and k are normed first.
template <bool IN16, bool OUT16, int VEC, bool PAGED, bool NORM>
__global__ void __launch_bounds__(kThreads) rope_heads_kernel(const HeadsParams p)
{
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int UPL = VEC > 1 ? 1 : 4;     // pieces (two runs) per lane: a head of 256 has 128 of 2 columns
    // Rounds whose loads are issued together, a batch ahead. (Two of runs of 8 instead of one took registers and with them warps: 26.9 us
    // instead of 25.9 for 8192 tokens x 32 heads of 128 in bf16; one of runs of 4 instead of two, 38.7 us instead of 35.3 from f32.)
    constexpr int BATCH = VEC == 4 ? 2 : 1;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t w = (uint64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const uint32_t token = (uint32_t)(w / p.splits), split = (uint32_t)(w - (uint64_t)token * p.splits);
    if (token >= p.tokens) return;
    const uint32_t lanes = p.lanes, at_once = 32 / lanes, sub = lane & (lanes - 1), group = lane / lanes;  // heads at once
    const uint32_t nq = p.heads[0], nkv = p.heads[1];
    const uint32_t units = p.dim / (2 * VEC), rot_units = p.rot / (2 * VEC), half = p.rot / 2;
    // A round is at_once heads of q, k or v.
    const uint32_t rounds_q = (nq + at_once - 1) / at_once, rounds_kv = (nkv + at_once - 1) / at_once, rounds = rounds_q + 2 * rounds_kv;

    uint32_t ca[UPL], cb[UPL];  // the first columns of this lane's runs
#pragma unroll
    for (int i = 0; i < UPL; ++i) {
        const uint32_t u = sub + i * 32;
        // Runs lie side by side over the lanes: of the two halves, whatever the pairs are. (Whole pairs in neighbouring runs read and wrote
        // half sectors.) Runs of one column: a pair.
        if (u < rot_units) {
            const bool pair = VEC == 1 && p.interleaved;
            ca[i] = pair ? 2 * u : VEC * u, cb[i] = pair ? 2 * u + 1 : half + VEC * u;
        } else {
            ca[i] = p.rot + VEC * (u - rot_units), cb[i] = ca[i] + (p.dim - p.rot) / 2;
        }
    }
    const size_t row_q = (size_t)token * p.src_stride[0], row_k = (size_t)token * p.src_stride[1], row_v = (size_t)token * p.src_stride[2];
    // Of a round: 0 q, 1 k, 2 v, and this lane's head among them.
    auto which = [&](uint32_t round, uint32_t &head) {
        const uint32_t kind = round < rounds_q ? 0u : round < rounds_q + rounds_kv ? 1u : 2u;
        head = (round - (kind == 0 ? 0 : kind == 1 ? rounds_q : rounds_q + rounds_kv)) * at_once + group;
        return kind;
    };
    using R = Run<IN16, VEC>;
    R ra[2][BATCH][UPL], rb[2][BATCH][UPL];
    auto fetch = [&](uint32_t round0, R (&a)[BATCH][UPL], R (&b)[BATCH][UPL]) {
#pragma unroll
        for (int y = 0; y < BATCH; ++y) {
            const uint32_t round = round0 + y * p.splits;
            if (round >= rounds) continue;
            uint32_t head;
            const uint32_t kind = which(round, head);
            if (head >= (kind == 0 ? nq : nkv)) continue;
            const void *src = kind == 0 ? p.src[0] : kind == 1 ? p.src[1] : p.src[2];
            const size_t row = (kind == 0 ? row_q : kind == 1 ? row_k : row_v) + head * p.dim;
#pragma unroll
            for (int i = 0; i < UPL; ++i)
                if (sub + i * 32 < units) a[y][i].load(src, row + ca[i]), b[y][i].load(src, row + cb[i]);
        }
    };
    fetch(split, ra[0], rb[0]);  // in flight while the position is found

    int32_t pos = 0;
    int64_t place = -1;  // of the token's row in the cache; -1: none
    if constexpr (PAGED) {
        const uint32_t s = paged::seq_of_row(p.seqs, token);
        if (s >= p.seqs.num_seqs) return;  // behind the last sequence
        const uint32_t len = paged::len_of(p.seqs, s), end = p.seqs.starts ? paged::start_of(p.seqs, s + 1) : s + 1;
        pos = (int32_t)(len - (end - token));  // below 0: in front of the sequence
        if (pos >= 0 && (uint64_t)pos < p.seqs.capacity) {
            const uint32_t page = (uint32_t)__ldcg(p.seqs.table + (size_t)s * p.seqs.max_pages + (uint32_t)pos / p.cache.page_size);
            if (page < p.cache.num_pages)
                place = (int64_t)(page * p.cache.page_stride + (uint64_t)((uint32_t)pos % p.cache.page_size) * p.cache.token_stride);
        }
    } else {
        pos = __ldcg(p.positions + token);
    }
    float2 turn[UPL][VEC];  // factor * (cos, sin) of this lane's pairs
    auto turn_at = [&](int i, uint32_t e) {
        uint32_t pair = (sub + i * 32) * VEC + e;
        if (VEC > 1 && p.interleaved) pair = (2 * e < VEC ? ca[i] + 2 * e : cb[i] + 2 * e - VEC) / 2;
        const uint64_t t = (uint64_t)(int64_t)pos * step_of(p.steps + pair);
        return turn_of((uint32_t)(t >> 32), p.factor);
    };
    // The heads that a warp has at once turn alike: their lanes work out a share each of the VEC pairs and hand them round. (Every lane
    // all of its own: half of the kernel's instructions.)
    auto turns = [&](auto shares) {
        constexpr int SHARES = decltype(shares)::value, EACH = VEC / SHARES;
        float2 own[UPL][EACH];
#pragma unroll
        for (int i = 0; i < UPL; ++i)
            if (sub + i * 32 < rot_units)
#pragma unroll
                for (int e = 0; e < EACH; ++e) own[i][e] = turn_at(i, SHARES > 1 ? group % SHARES * EACH + e : e);
#pragma unroll
        for (int i = 0; i < UPL; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                turn[i][e] = own[i][e % EACH];
                if (SHARES > 1) {
                    turn[i][e].x = __shfl_sync(0xffffffffu, turn[i][e].x, sub + lanes * (e / EACH));
                    turn[i][e].y = __shfl_sync(0xffffffffu, turn[i][e].y, sub + lanes * (e / EACH));
                }
            }
    };
    if (VEC >= 4 && at_once >= 4) turns(std::integral_constant<int, VEC >= 4 ? 4 : 1>{});
    else if (VEC >= 4 && at_once == 2) turns(std::integral_constant<int, VEC >= 4 ? 2 : 1>{});
    else turns(std::integral_constant<int, 1>{});
    float wq[UPL][2 * VEC], wk[UPL][2 * VEC];  // 1 + the norms' weights of this lane's columns
    if constexpr (NORM) {
        auto load = [](const float *at) {
            float v;
            asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(at) : "memory");  // not before the wait above
            return 1.0f + v;
        };
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
            if (sub + i * 32 >= units) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                wq[i][e] = load(p.norm_w[0] + ca[i] + e), wq[i][VEC + e] = load(p.norm_w[0] + cb[i] + e);
                wk[i][e] = load(p.norm_w[1] + ca[i] + e), wk[i][VEC + e] = load(p.norm_w[1] + cb[i] + e);
            }
        }
    }

    auto process = [&](uint32_t round0, const R (&ia)[BATCH][UPL], const R (&ib)[BATCH][UPL]) {
#pragma unroll
        for (int y = 0; y < BATCH; ++y) {
            const uint32_t round = round0 + y * p.splits;
            if (round >= rounds) continue;
            uint32_t head;
            const uint32_t kind = which(round, head);
            const bool there = head < (kind == 0 ? nq : nkv) && (kind == 0 || place >= 0);
            float a[UPL][VEC], b[UPL][VEC];
#pragma unroll
            for (int i = 0; i < UPL; ++i) ia[y][i].get(a[i]), ib[y][i].get(b[i]);
            if (NORM && kind < 2) {  // the whole warp: heads that are not there are summed for nothing
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < UPL; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e)
                        if (sub + i * 32 < units) ss = fmaf(a[i][e], a[i][e], ss), ss = fmaf(b[i][e], b[i][e], ss);
                for (uint32_t o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)p.dim) + p.eps));
#pragma unroll
                for (int i = 0; i < UPL; ++i)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        a[i][e] = __fmul_rn(__fmul_rn(a[i][e], inv), kind == 0 ? wq[i][e] : wk[i][e]);
                        b[i][e] = __fmul_rn(__fmul_rn(b[i][e], inv), kind == 0 ? wq[i][VEC + e] : wk[i][VEC + e]);
                    }
            }
            if (!there) continue;
#pragma unroll
            for (int i = 0; i < UPL; ++i) {
                const uint32_t u = sub + i * 32;
                if (u >= units) continue;
                if (kind < 2 && u < rot_units) {
                    if (VEC == 1 || !p.interleaved) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float2 cs = turn[i][e];
                            const float x = a[i][e], z = b[i][e];
                            a[i][e] = x * cs.x - z * cs.y, b[i][e] = x * cs.y + z * cs.x;
                        }
                    } else {
                        constexpr int H = VEC / 2;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float2 cs = turn[i][e];
                            float &x = e < H ? a[i][(2 * e) % VEC] : b[i][(2 * e) % VEC], &z = e < H ? a[i][(2 * e + 1) % VEC] : b[i][(2 * e + 1) % VEC];
                            const float x0 = x, z0 = z;
                            x = x0 * cs.x - z0 * cs.y, z = x0 * cs.y + z0 * cs.x;
                        }
                    }
                }
                if (!PAGED || kind == 0) {
                    const size_t row = (size_t)token * p.out_stride + head * p.dim;
                    store_run<OUT16, VEC>(p.out, row + ca[i], a[i]), store_run<OUT16, VEC>(p.out, row + cb[i], b[i]);
                } else {
                    const size_t row = (size_t)place + head * p.cache.head_stride;
                    uint16_t *dst = kind == 1 ? p.cache.k : p.cache.v;
                    store_run<true, VEC>(dst, row + ca[i], a[i]), store_run<true, VEC>(dst, row + cb[i], b[i]);
                }
            }
        }
    };
    for (uint32_t round = split; round < rounds; round += 2 * BATCH * p.splits) {
        fetch(round + BATCH * p.splits, ra[1], rb[1]);
        process(round, ra[0], rb[0]);
        fetch(round + 2 * BATCH * p.splits, ra[0], rb[0]);
        process(round + BATCH * p.splits, ra[1], rb[1]);
    }
}

/// `run`: the columns of a run, 8, 4 or 1.
template <bool PAGED>
Result launch_heads(TesslRuntime *rt, const char *what, HeadsParams p, bool in16, bool out16, uint32_t run)
{
    p.lanes = 32;
    if (run > 1)
        while (p.lanes > 1 && p.lanes / 2 * 2 * run >= p.dim) p.lanes /= 2;
    // The heads of few tokens are spread over several warps, until there are 16 for each SM.
    const uint32_t at_once = 32 / p.lanes, rounds = (p.heads[0] + at_once - 1) / at_once + 2 * ((p.heads[1] + at_once - 1) / at_once);
    p.splits = std::min(rounds, std::max(1u, 16 * (uint32_t)rt->sm_count / p.tokens));
    const uint64_t blocks = ((uint64_t)p.tokens * p.splits - 1) / (kThreads / 32) + 1;  // below 2^31: p.tokens is
    auto go = [&](auto kernel) { return launch_pdl(rt, what, kernel, dim3((unsigned)blocks), dim3(kThreads), 0, p); };
    auto typed = [&](auto in, auto out, auto norm) {
        constexpr bool IN = decltype(in)::value, OUT = decltype(out)::value, NORM = decltype(norm)::value;
        if constexpr (IN)
            if (run == 8) return go(rope_heads_kernel<IN, OUT, 8, PAGED, NORM>);
        return run > 1 ? go(rope_heads_kernel<IN, OUT, 4, PAGED, NORM>) : go(rope_heads_kernel<IN, OUT, 1, PAGED, NORM>);
    };
    const std::true_type yes{};
    const std::false_type no{};
    if constexpr (PAGED) {
        if (p.norm_w[0]) return in16 ? typed(yes, yes, yes) : typed(no, yes, yes);
        return in16 ? typed(yes, yes, no) : typed(no, yes, no);
    } else {
        if (in16) return out16 ? typed(yes, yes, no) : typed(yes, no, no);
        return out16 ? typed(no, yes, no) : typed(no, no, no);
    }
}

Result rope_validate(const TesslRope &r, uint32_t head_dim, const char *what)
{
    if (r.rot_dim % 2 != 0 || r.rot_dim > head_dim) return fmt("%s: rot_dim %u is odd or more than head_dim %u", what, r.rot_dim, head_dim);
    if (!std::isfinite(r.factor)) return fmt("%s: the rope's factor is not finite", what);
    TESSL_TRY(require(r.steps, r.rot_dim / 2, 8, What(what) + " rope steps"));
    if (((uintptr_t)r.steps.ptr & 7u) != 0) return fmt("%s: rope steps must be 8-byte aligned", what);
    return ok();
}

/// Columns of the longest run that memory of 16-bit or 32-bit values allows: 8, 4 or 1.
uint32_t run_of(const void *p, uint32_t stride, bool is16)
{
    const uint32_t size = is16 ? 2 : 4;
    for (uint32_t run : {8u, 4u})
        if (((uintptr_t)p & (std::min(run * size, 16u) - 1)) == 0 && stride % (std::min(run * size, 16u) / size) == 0) return run;
    return 1;
}

/// The same of a head: whole runs, two by two, in its rotated part and behind it; 8 columns of f32 are two loads, no better than 4.
uint32_t run_of(uint32_t dim, uint32_t rot, bool in16)
{
    if (in16 && dim % 16 == 0 && rot % 16 == 0) return 8;
    return dim % 8 == 0 && rot % 8 == 0 ? 4 : 1;
}

}  // namespace

namespace nn {

Result rope_steps(uint32_t rot_dim, double theta, const TesslRopeScaling *scaling, uint64_t *steps, float *factor)
{
    const char *what = "rope_steps";
    if (rot_dim % 2 != 0 || rot_dim > 2 * kMaxPairs) return fmt("%s: rot_dim %u is odd or more than %u", what, rot_dim, 2 * kMaxPairs);
    if (!(theta > 1.0) || !std::isfinite(theta)) return fmt("%s: theta must be finite and more than 1", what);
    if (!factor || (!steps && rot_dim)) return fmt("%s: null output", what);
    TesslRopeScaling s{};
    if (scaling) s = *scaling;
    if (s.kind > TESSL_ROPE_SCALE_YARN) return fmt("%s: unknown scaling %u", what, s.kind);
    if (s.kind == TESSL_ROPE_SCALE_NONE) s.factor = 1.0;
    if (!(s.factor >= 1.0) || !std::isfinite(s.factor)) return fmt("%s: the scaling's factor must be finite and at least 1", what);
    const bool by_wave = s.kind == TESSL_ROPE_SCALE_WAVELENGTH, yarn = s.kind == TESSL_ROPE_SCALE_YARN;
    if (s.low == 0.0) s.low = 1.0;
    if (s.high == 0.0) s.high = yarn ? 32.0 : 4.0;
    if (by_wave || yarn) {
        if (!(s.original > 0.0) || !std::isfinite(s.original)) return fmt("%s: the scaling needs the trained context's length", what);
        if (!(s.low > 0.0) || !(s.high > s.low) || !std::isfinite(s.high)) return fmt("%s: the scaling's low and high must be positive and ascending", what);
    }
    const long double two_pi = 6.283185307179586476925286766559005768L;
    long double base = theta;
    if (s.kind == TESSL_ROPE_SCALE_NTK && rot_dim > 2) base = theta * std::pow((long double)s.factor, (long double)rot_dim / (rot_dim - 2));
    long double ramp_lo = 0, ramp_hi = 1;
    if (yarn) {  // the pairs that turn so many times within the trained context
        ramp_lo = std::max(std::floor(rot_dim * std::log(s.original / (s.high * two_pi)) / (2 * std::log(base))), 0.0L);
        ramp_hi = std::min(std::ceil(rot_dim * std::log(s.original / (s.low * two_pi)) / (2 * std::log(base))), (long double)rot_dim - 1);
    }
    for (uint32_t i = 0; i < rot_dim / 2; ++i) {
        long double w = std::pow(base, -2.0L * i / rot_dim);
        if (s.kind == TESSL_ROPE_SCALE_LINEAR) w /= s.factor;
        if (by_wave) {
            const long double turns = s.original * w / two_pi;
            const long double keep = std::min(1.0L, std::max(0.0L, (turns - s.low) / (s.high - s.low)));
            w = keep * w + (1.0L - keep) * (w / s.factor);
        }
        if (yarn) {
            const long double ramp = std::min(1.0L, std::max(0.0L, (i - ramp_lo) / std::max(ramp_hi - ramp_lo, 0.001L)));
            w = (w / s.factor) * ramp + w * (1.0L - ramp);
        }
        const long double step = std::floor(w / two_pi * 0x1p64L + 0.5L);  // w <= 1: below 2^62
        steps[i] = (uint64_t)step;
    }
    *factor = yarn && s.factor > 1.0 ? (float)(0.1 * std::log(s.factor) + 1.0) : 1.0f;
    return ok();
}

Result rope(TesslRuntime *rt, const TesslBuf &x, const TesslBuf &positions, const TesslBuf &out, const TesslRope &rope, uint32_t tokens,
            uint32_t n_heads, uint32_t head_dim, uint32_t x_stride, uint32_t out_stride, bool x_as_bf16, bool out_as_bf16)
{
    const char *what = "rope";
    if (head_dim == 0 || head_dim % 2 != 0 || head_dim > 2 * kMaxPairs) return fmt("%s: head_dim %u is not even and up to %u", what, head_dim, 2 * kMaxPairs);
    TESSL_TRY(rope_validate(rope, head_dim, what));
    if (tokens > 0x7fffffffu) return fmt("%s: too many tokens", what);
    if (n_heads > (1u << 20)) return fmt("%s: too many heads", what);
    const uint64_t width = elems(n_heads, head_dim);
    TESSL_TRY(paged::rows_validate(x, tokens, width, &x_stride, x_as_bf16 ? 2 : 4, what, "x"));
    TESSL_TRY(paged::rows_validate(out, tokens, width, &out_stride, out_as_bf16 ? 2 : 4, what, "out"));
    TESSL_TRY(require(positions, tokens, 4, "rope positions"));
    if (((uintptr_t)positions.ptr & 3u) != 0) return fmt("%s: positions must be 4-byte aligned", what);
    if (tokens == 0 || n_heads == 0) return ok();
    const Named writes[] = {{"out", &out}};
    const Named reads[] = {{"positions", &positions}, {"rope steps", &rope.steps}, {"x", &x}};
    // out may be x itself: every value is read and written by the same thread
    const bool in_place = out.ptr == x.ptr && x_as_bf16 == out_as_bf16 && x_stride == out_stride;
    TESSL_TRY(require_disjoint_writes(what, writes, 1, reads, in_place ? 2 : 3));
    HeadsParams p{};
    p.src[0] = x.ptr, p.src_stride[0] = x_stride, p.heads[0] = n_heads;
    p.out = out.ptr, p.out_stride = out_stride;
    p.positions = static_cast<const int32_t *>(positions.ptr), p.steps = static_cast<const uint64_t *>(rope.steps.ptr);
    p.factor = rope.factor, p.tokens = tokens, p.dim = head_dim, p.rot = rope.rot_dim, p.interleaved = rope.interleaved != 0;
    const uint32_t run = std::min({run_of(head_dim, rope.rot_dim, x_as_bf16), run_of(x.ptr, x_stride, x_as_bf16), run_of(out.ptr, out_stride, out_as_bf16)});
    return launch_heads<false>(rt, "rope launch", p, x_as_bf16, out_as_bf16, run);
}

Result kv_append_paged(TesslRuntime *rt, const TesslBuf &q, const TesslBuf &k, const TesslBuf &v, const TesslBuf &q_out,
                       const TesslPagedKv &cache, const TesslPagedSeqs &seqs, const TesslRope *rope, const TesslQkNorm *norm,
                       uint32_t total_new, uint32_t n_heads, uint32_t q_stride, uint32_t k_stride, uint32_t v_stride, bool in_as_bf16)
{
    const char *what = "kv_append_paged";
    HeadsParams p{};
    TESSL_TRY(paged::cache_validate(cache, what, &p.cache));
    TESSL_TRY(paged::seqs_validate(seqs, cache, total_new, what, &p.seqs));
    const uint32_t dim = cache.head_dim;
    const size_t elem = in_as_bf16 ? 2 : 4;
    if (n_heads > (1u << 20)) return fmt("%s: too many heads", what);
    if (rope) TESSL_TRY(rope_validate(*rope, dim, what));
    if (norm) {
        if (!(norm->eps > 0.0f) || !(norm->eps < 3.0e38f)) return fmt("%s: eps must be finite and positive", what);
        if (n_heads) TESSL_TRY(require(norm->q_weight, dim, 4, "kv_append_paged q norm weight"));
        TESSL_TRY(require(norm->k_weight, dim, 4, "kv_append_paged k norm weight"));
        if ((((uintptr_t)norm->q_weight.ptr | (uintptr_t)norm->k_weight.ptr) & 3u) != 0) return fmt("%s: norm weights must be 4-byte aligned", what);
    }
    if (n_heads) {
        TESSL_TRY(paged::rows_validate(q, total_new, elems(n_heads, dim), &q_stride, elem, what, "q"));
        uint32_t out_stride = 0;
        TESSL_TRY(paged::rows_validate(q_out, total_new, elems(n_heads, dim), &out_stride, 2, what, "q_out"));
        p.out_stride = out_stride;
    }
    TESSL_TRY(paged::rows_validate(k, total_new, elems(cache.n_kv_heads, dim), &k_stride, elem, what, "k"));
    TESSL_TRY(paged::rows_validate(v, total_new, elems(cache.n_kv_heads, dim), &v_stride, elem, what, "v"));
    const TesslBuf none{nullptr, 0};
    const Named writes[] = {{"cache k", &cache.k}, {"cache v", &cache.v}, {"q_out", n_heads ? &q_out : &none}};
    const Named reads[] = {{"q", n_heads ? &q : &none}, {"k", &k}, {"v", &v}, {"page_table", &seqs.page_table}, {"kv_lens", &seqs.kv_lens},
                           {"q_starts", &seqs.q_starts}, {"rope steps", rope ? &rope->steps : &none},
                           {"q norm weight", norm ? &norm->q_weight : &none}, {"k norm weight", norm ? &norm->k_weight : &none}};
    TESSL_TRY(require_disjoint_writes(what, writes, 3, reads, 9));
    if (total_new == 0) return ok();
    p.src[0] = q.ptr, p.src[1] = k.ptr, p.src[2] = v.ptr;
    p.src_stride[0] = q_stride, p.src_stride[1] = k_stride, p.src_stride[2] = v_stride;
    p.heads[0] = n_heads, p.heads[1] = cache.n_kv_heads;
    p.out = q_out.ptr, p.tokens = total_new, p.dim = dim;
    if (rope) p.steps = static_cast<const uint64_t *>(rope->steps.ptr), p.factor = rope->factor, p.rot = rope->rot_dim, p.interleaved = rope->interleaved != 0;
    if (norm) {
        p.norm_w[1] = static_cast<const float *>(norm->k_weight.ptr);
        p.norm_w[0] = n_heads ? static_cast<const float *>(norm->q_weight.ptr) : p.norm_w[1];
        p.eps = norm->eps;
    }
    uint32_t run = std::min({run_of(dim, p.rot, in_as_bf16), run_of(k.ptr, k_stride, in_as_bf16), run_of(v.ptr, v_stride, in_as_bf16)});
    if (n_heads) run = std::min({run, run_of(q.ptr, q_stride, in_as_bf16), run_of(q_out.ptr, p.out_stride, true)});
    return launch_heads<true>(rt, "kv_append_paged launch", p, in_as_bf16, true, run);
}

}  // namespace nn
}  // namespace tessl
