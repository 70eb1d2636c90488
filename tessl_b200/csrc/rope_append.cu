// Rotary positions, and the append of new keys and values to a paged cache with the rotation (and the heads' norm) on the way.
//
// Pair i of a head turns by position * w_i radians. The angle is kept in turns as a 64-bit fraction: steps[i] =
// round(2^64 w_i / 2 pi), and position * steps[i] modulo 2^64 is the angle modulo one turn with an error below position * 2^-65 turns,
// for any 32-bit position. (position * w_i in f32 is off by 0.06 radians at position 10^6.) Sine and cosine of pi times a
// fraction in [-1, 1) follow in f32.
//
// One kernel for both operators: a token's heads are spread over groups of lanes, a lane holds two runs of four columns of a head,
// which are the two halves of four pairs or four whole ones, so a rotation needs no exchange and the norm one butterfly.
// The angles are computed once per token and shared by its heads. Bound by memory from some thousand tokens on, by the
// chain offset -> length -> page id -> store (four round trips to L2) below.
#include <algorithm>
#include <cmath>

#include "paged_common.cuh"

namespace tessl {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxTokens = 8;   // tokens per block, at most: one per warp
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
    uint32_t lanes;             // per head, a power of two
    uint32_t tokens_per_block;  // a power of two
    uint32_t splits;            // blocks that share the heads of a token
};

template <bool IN16, int VEC>
struct Piece {  // two runs of VEC columns
    float a[VEC], b[VEC];
};

template <bool IN16, int VEC>
__device__ __forceinline__ void load_run(const void *src, size_t at, float (&v)[VEC])
{
    if constexpr (VEC == 4 && IN16) {
        const uint2 w = dev::ld_after_wait8(static_cast<const uint16_t *>(src) + at);
        v[0] = dev::bf16_lo(w.x), v[1] = dev::bf16_hi(w.x), v[2] = dev::bf16_lo(w.y), v[3] = dev::bf16_hi(w.y);
    } else if constexpr (VEC == 4) {
        const uint4 w = dev::ld_after_wait16(static_cast<const float *>(src) + at);
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    } else if constexpr (IN16) {
        v[0] = __uint_as_float((uint32_t)__ldcg(static_cast<const unsigned short *>(src) + at) << 16);
    } else {
        v[0] = __ldcg(static_cast<const float *>(src) + at);
    }
}

/// Two f32 -> a bf16 pair, to nearest even.
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

template <bool OUT16, int VEC>
__device__ __forceinline__ void store_run(void *dst, size_t at, const float (&v)[VEC])
{
    if constexpr (VEC == 4 && OUT16) {
        *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(dst) + at) = make_uint2(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]));
    } else if constexpr (VEC == 4) {
        *reinterpret_cast<float4 *>(static_cast<float *>(dst) + at) = make_float4(v[0], v[1], v[2], v[3]);
    } else if constexpr (OUT16) {
        static_cast<uint16_t *>(dst)[at] = (uint16_t)bf16_pair(v[0], 0.0f);
    } else {
        static_cast<float *>(dst)[at] = v[0];
    }
}

/// VEC = 4: rot a multiple of 8 and everything aligned for whole runs. VEC = 1: anything else, 32 lanes per head.
/// PAGED: rows find their sequence, positions come from the lengths, k and v go to the cache; else positions are given.
template <bool IN16, bool OUT16, int VEC, bool PAGED>
__global__ void __launch_bounds__(kThreads) rope_heads_kernel(const HeadsParams p)
{
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int UPL = VEC == 4 ? 1 : 4;  // pieces per lane: a head of 256 has 32 of 8 columns, 128 of 2
    __shared__ float2 turn[kMaxTokens][kMaxPairs];  // factor * (cos, sin)
    __shared__ int64_t place[kMaxTokens];           // of the token's row in the cache; -1: none
    __shared__ uint32_t live[kMaxTokens];           // the row belongs to a sequence
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t tpb = p.tokens_per_block, t0 = blockIdx.x * tpb;
    const uint32_t lanes = p.lanes, groups = kThreads / lanes, group = tid / lanes, sub = tid & (lanes - 1);
    const uint32_t nq = p.heads[0], nkv = p.heads[1], nh = nq + 2 * nkv;  // heads of a token
    const uint32_t units = p.dim / (2 * VEC), rot_units = p.rot / (2 * VEC), half = p.rot / 2;
    // Work item w of the block's share: head w % nh of token w / nh.
    const uint32_t items = tpb * nh, first = blockIdx.y * groups + group, step = groups * p.splits;

    auto columns = [&](uint32_t u, uint32_t &a, uint32_t &b) {  // the two runs of piece u
        if (u < rot_units) {
            a = p.interleaved ? 2 * VEC * u : VEC * u;
            b = p.interleaved ? a + VEC : half + a;
        } else {
            a = p.rot + 2 * VEC * (u - rot_units), b = a + VEC;
        }
    };
    auto which = [&](uint32_t head, uint32_t &h) {  // 0 q, 1 k, 2 v; h: the head among them
        if (head < nq) return h = head, 0u;
        h = head - nq;
        if (h < nkv) return 1u;
        h -= nkv;
        return 2u;
    };
    Piece<IN16, VEC> cur[UPL];
    auto fetch = [&](uint32_t w, Piece<IN16, VEC> (&v)[UPL]) {
        const uint32_t token = t0 + w / nh;
        uint32_t h;
        const uint32_t kind = which(w % nh, h);
        if (token >= p.tokens) return;
        const void *src = kind == 0 ? p.src[0] : kind == 1 ? p.src[1] : p.src[2];
        const size_t row = (size_t)token * (kind == 0 ? p.src_stride[0] : kind == 1 ? p.src_stride[1] : p.src_stride[2]) + (size_t)h * p.dim;
#pragma unroll
        for (int i = 0; i < UPL; ++i) {
            const uint32_t u = sub + i * 32;
            if (u >= units) continue;
            uint32_t a, b;
            columns(u, a, b);
            load_run<IN16, VEC>(src, row + a, v[i].a), load_run<IN16, VEC>(src, row + b, v[i].b);
        }
    };
    if (first < items) fetch(first, cur);  // in flight while the positions are found

    {   // warp w looks after token w % tpb, with the other warps of that token a share of its angles
        const uint32_t tl = warp & (tpb - 1), row = t0 + tl, share = kThreads / 32 / tpb;
        int32_t pos = 0;
        bool alive = row < p.tokens;
        if (PAGED && alive) {
            const uint32_t s = paged::seq_of_row(p.seqs, row);
            alive = s < p.seqs.num_seqs;
            if (alive) {
                const uint32_t len = paged::len_of(p.seqs, s), end = p.seqs.starts ? paged::start_of(p.seqs, s + 1) : s + 1;
                pos = (int32_t)(len - (end - row));  // below 0: in front of the sequence
                if (lane == 0 && warp < tpb) {
                    int64_t at = -1;
                    if (pos >= 0 && (uint64_t)pos < p.seqs.capacity) {
                        const uint32_t page = (uint32_t)__ldcg(p.seqs.table + (size_t)s * p.seqs.max_pages + (uint32_t)pos / p.cache.page_size);
                        if (page < p.cache.num_pages)
                            at = (int64_t)(page * p.cache.page_stride + (uint64_t)((uint32_t)pos % p.cache.page_size) * p.cache.token_stride);
                    }
                    place[tl] = at;
                }
            }
        } else if (alive) {
            pos = __ldcg(p.positions + row);
        }
        if (lane == 0 && warp < tpb) live[tl] = alive;
        for (uint32_t i = (warp / tpb) * 32 + lane; i < half && alive; i += share * 32) {
            const uint64_t t = (uint64_t)(int64_t)pos * __ldcg(reinterpret_cast<const unsigned long long *>(p.steps) + i);
            float s, c;
            sincospif(__ll2float_rn((long long)t) * 0x1p-63f, &s, &c);
            turn[tl][i] = make_float2(p.factor * c, p.factor * s);
        }
    }
    __syncthreads();

    for (uint32_t w = first; w < items; w += step) {
        Piece<IN16, VEC> next[UPL];
        if (w + step < items) fetch(w + step, next);
        const uint32_t tl = w / nh, token = t0 + tl;
        uint32_t h;
        const uint32_t kind = which(w % nh, h);
        const bool alive = token < p.tokens && live[tl];
        if (PAGED && kind < 2 && p.norm_w[0]) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < UPL; ++i)
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if (sub + i * 32 < units) ss = fmaf(cur[i].a[e], cur[i].a[e], ss), ss = fmaf(cur[i].b[e], cur[i].b[e], ss);
            const uint32_t mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1u) << (lane & ~(lanes - 1));
            for (uint32_t o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
            const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)p.dim) + p.eps));
            const float *nw = kind == 0 ? p.norm_w[0] : p.norm_w[1];
#pragma unroll
            for (int i = 0; i < UPL; ++i) {
                const uint32_t u = sub + i * 32;
                if (u >= units) continue;
                uint32_t a, b;
                columns(u, a, b);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    cur[i].a[e] = __fmul_rn(__fmul_rn(cur[i].a[e], inv), 1.0f + __ldcg(nw + a + e));
                    cur[i].b[e] = __fmul_rn(__fmul_rn(cur[i].b[e], inv), 1.0f + __ldcg(nw + b + e));
                }
            }
        }
        const int64_t at = PAGED ? place[tl] : 0;
        if (alive && (kind == 0 || at >= 0)) {
#pragma unroll
            for (int i = 0; i < UPL; ++i) {
                const uint32_t u = sub + i * 32;
                if (u >= units) continue;
                uint32_t a, b;
                columns(u, a, b);
                Piece<IN16, VEC> &c = cur[i];
                if (kind < 2 && u < rot_units) {
                    if (VEC == 1 || !p.interleaved) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float2 cs = turn[tl][u * VEC + e];
                            const float x = c.a[e], y = c.b[e];
                            c.a[e] = x * cs.x - y * cs.y, c.b[e] = x * cs.y + y * cs.x;
                        }
                    } else {
                        constexpr int H = VEC / 2;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float2 cs = turn[tl][u * VEC + e];
                            float &x = e < H ? c.a[(2 * e) % VEC] : c.b[(2 * e) % VEC], &y = e < H ? c.a[(2 * e + 1) % VEC] : c.b[(2 * e + 1) % VEC];
                            const float x0 = x, y0 = y;
                            x = x0 * cs.x - y0 * cs.y, y = x0 * cs.y + y0 * cs.x;
                        }
                    }
                }
                if (!PAGED || kind == 0) {
                    const size_t row = (size_t)token * p.out_stride + (size_t)h * p.dim;
                    store_run<OUT16, VEC>(p.out, row + a, c.a), store_run<OUT16, VEC>(p.out, row + b, c.b);
                } else {
                    const size_t row = (size_t)at + (size_t)h * p.cache.head_stride;
                    uint16_t *dst = kind == 1 ? p.cache.k : p.cache.v;
                    store_run<true, VEC>(dst, row + a, c.a), store_run<true, VEC>(dst, row + b, c.b);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < UPL; ++i) cur[i] = next[i];
    }
}

template <bool PAGED>
Result launch_heads(TesslRuntime *rt, const char *what, HeadsParams p, bool in16, bool out16, bool wide)
{
    const uint32_t nh = p.heads[0] + 2 * p.heads[1];
    p.lanes = 32;
    if (wide)
        while (p.lanes > 1 && p.lanes / 2 * 8 >= p.dim) p.lanes /= 2;
    const uint32_t groups = kThreads / p.lanes;
    // Tokens of few heads share a block; the heads of few tokens are spread over several, until there is a block for each SM.
    p.tokens_per_block = 1;
    while (p.tokens_per_block < kMaxTokens && p.tokens_per_block * 2 * nh <= groups &&
           p.tokens / (p.tokens_per_block * 2) >= (uint32_t)rt->sm_count)
        p.tokens_per_block *= 2;
    const uint32_t blocks = (p.tokens - 1) / p.tokens_per_block + 1, rounds = (p.tokens_per_block * nh - 1) / groups + 1;
    p.splits = min(min(rounds, 65535u), max(1u, 2 * (uint32_t)rt->sm_count / blocks));
    auto go = [&](auto kernel) { return launch_pdl(rt, what, kernel, dim3(blocks, p.splits), dim3(kThreads), 0, p); };
    if (PAGED) {
        if (wide) return in16 ? go(rope_heads_kernel<true, true, 4, PAGED>) : go(rope_heads_kernel<false, true, 4, PAGED>);
        return in16 ? go(rope_heads_kernel<true, true, 1, PAGED>) : go(rope_heads_kernel<false, true, 1, PAGED>);
    }
    if (wide) {
        if (in16) return out16 ? go(rope_heads_kernel<true, true, 4, PAGED>) : go(rope_heads_kernel<true, false, 4, PAGED>);
        return out16 ? go(rope_heads_kernel<false, true, 4, PAGED>) : go(rope_heads_kernel<false, false, 4, PAGED>);
    }
    if (in16) return out16 ? go(rope_heads_kernel<true, true, 1, PAGED>) : go(rope_heads_kernel<true, false, 1, PAGED>);
    return out16 ? go(rope_heads_kernel<false, true, 1, PAGED>) : go(rope_heads_kernel<false, false, 1, PAGED>);
}

Result rope_validate(const TesslRope &r, uint32_t head_dim, const char *what)
{
    if (r.rot_dim % 2 != 0 || r.rot_dim > head_dim) return fmt("%s: rot_dim %u is odd or more than head_dim %u", what, r.rot_dim, head_dim);
    if (!std::isfinite(r.factor)) return fmt("%s: the rope's factor is not finite", what);
    TESSL_TRY(require(r.steps, r.rot_dim / 2, 8, What(what) + " rope steps"));
    if (((uintptr_t)r.steps.ptr & 7u) != 0) return fmt("%s: rope steps must be 8-byte aligned", what);
    return ok();
}

bool aligned(const void *p, uint32_t stride, bool is16)
{
    return ((uintptr_t)p & (is16 ? 7u : 15u)) == 0 && stride % 4 == 0;
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
    const bool wide = head_dim % 8 == 0 && rope.rot_dim % 8 == 0 && aligned(x.ptr, x_stride, x_as_bf16) && aligned(out.ptr, out_stride, out_as_bf16);
    return launch_heads<false>(rt, "rope launch", p, x_as_bf16, out_as_bf16, wide);
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
    bool wide = p.rot % 8 == 0 && aligned(k.ptr, k_stride, in_as_bf16) && aligned(v.ptr, v_stride, in_as_bf16);
    if (n_heads) wide = wide && aligned(q.ptr, q_stride, in_as_bf16) && aligned(q_out.ptr, p.out_stride, true);
    return launch_heads<true>(rt, "kv_append_paged launch", p, in_as_bf16, true, wide);
}

}  // namespace nn
}  // namespace tessl
