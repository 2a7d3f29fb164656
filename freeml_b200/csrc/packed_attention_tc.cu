// Causal attention over packed prompts with grouped heads, fp16 and bf16, on
// the tensor cores: S = Q K^T * scale with the causal mask, row softmax, P V,
// as one pass over the keys with a running maximum and sum.
//
// CTA = 12 warps on two tiles, A and B, of 128 query rows of one key/value
// head (packed.cuh: tokens in order and, for each, the query heads of the
// group, so that a group shares every key and value tile).  The two tiles'
// phases interleave: the tensor cores work on one while the other's softmax
// runs.
//   warps 0-3, 4-7  softmax of tile A, B (thread = TMEM lane = query row)
//   warps 8, 9      tile A's / B's tcgen05.mma (one lane elected)
//   warp 10         one thread issues every TMA copy; the warp then zeroes the
//                   rows past the sequence's end in its last value tile
//                   (another sequence's rows, or its NaN, lie there)
//   warp 11         idle: registers are shared out by groups of four warps
// Keys and values are copied 128 rows at a time and used in halves of 64.  TMEM,
// per query tile: two score buffers of 64 fp32 columns, S of half i in buffer
// i % 2, overwritten in place by P in 16 bits (32 columns, the A operand of
// O += P V, read from TMEM), and the output's hd columns, which stay there over
// all keys.  With two buffers S of half i + 1 is there before P of half i is, and
// the softmax warps never wait for a product in the steady state; one buffer of
// 128 keys costs the tensor cores less (an S product of 64 keys takes 3/4 of the
// time of one of 128) but took 4640 cycles for 128 keys and 256 rows of head
// dim 128, against 3950.
// A row rescales its output only when a score rises by more than 2^8 (bf16:
// 2^40) over the maximum that its P is taken against; fp16 P is taken 2^7
// larger, so that it uses the type's range (at most 2^15) and small
// probabilities stay above its smallest numbers.
//
// What bounds it: per 128 keys and 256 rows of head dim 128, the products take
// 2560 cycles of the tensor cores and the exponentials 2048 of the special
// function units.
// Every wait is bounded and returns early once any role has recorded an expiry.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "f32x2.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace fml {

__device__ int g_packed_tc_timeouts;

namespace {

constexpr int THREADS = 12 * 32;
constexpr int KT = 128;  // keys of a copied tile
constexpr int KH = 64;   // keys of a half: one S and one P product

template <int HD>
struct Shape
{
    static constexpr int COLS = HD < 64 ? HD : 64;      // columns of a box: a row of 64 or 128 bytes
    static constexpr int BOXES = HD / COLS;
    static constexpr uint32_t ROW = COLS * 2;
    static constexpr uint32_t BOX = 128 * ROW;          // 128 rows of a box
    static constexpr uint32_t TILE = BOXES * BOX;       // a Q, K or V tile
    static constexpr int STAGES = HD == 128 ? 2 : 4;
    static constexpr uint32_t SMEM = 2 * TILE + 2 * STAGES * TILE + 1024 + 512;
    // TMEM columns of tile x: S / P buffers 0 and 1, the output
    static constexpr uint32_t TX = 256, O = 2 * KH;
    // shared-memory operand descriptors: 8-row groups of the swizzled rows
    static constexpr uint64_t LAYOUT = HD < 64 ? 4ull << 61 : 2ull << 61;  // 64- or 128-byte swizzle
    static constexpr uint64_t SBO = (uint64_t)(8 * ROW >> 4) << 32;
    static constexpr uint64_t KDESC = LAYOUT | SBO | (1ull << 16) | (1ull << 46);
    // value tile as an N-major operand: the next columns a box on, the next 8 keys a row group on
    static constexpr uint64_t VDESC = LAYOUT | SBO | ((uint64_t)(BOX >> 4) << 16) | (1ull << 46);
};

// per query tile x: S and P by buffer (2 x + buffer), the output, the end; per
// stage: K and V copies landed, K and V consumed by each query tile
enum Bar { B_QF, B_VR, B_S0, B_P0 = B_S0 + 4, B_O0 = B_P0 + 4, B_FIN = B_O0 + 2, B_KF = B_FIN + 2 };
template <int ST>
struct Bars
{
    static constexpr int KF = B_KF, VF = KF + ST, KE = VF + ST, VE = KE + 2 * ST, N = VE + 2 * ST;
};

template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int M, int N)
{
    const uint32_t f = std::is_same_v<T, __half> ? 0u : 1u;
    return (1u << 4) | (f << 7) | (f << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// Products and commits are issued by a whole warp, of which the hardware elects
// one lane: its operands are then the same in the warp for the compiler too.
// From a branch of one thread a product costs 80 to 130 cycles to issue, more
// than it takes; so, 15 to 25.
__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

__device__ __forceinline__ void commit(uint64_t* bar)
{
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc::smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(tc::smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Scores `first` .. of 32 columns, where a mask bites, to -inf (a select: NaN may lie there).
__device__ __forceinline__ void mask32(uint32_t (&u)[32], bool masked, int first)
{
    if (masked)
    {
#pragma unroll
        for (int i = 0; i < 32; ++i) u[i] = i < first ? u[i] : 0xff800000u;
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if constexpr (std::is_same_v<T, __half>)
    {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    else
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

}  // namespace

template <typename T, int HD>
__global__ void __launch_bounds__(THREADS, 1) packed_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                         const __grid_constant__ CUtensorMap map_k,
                                                                         const __grid_constant__ CUtensorMap map_v,
                                                                         T* __restrict__ out, PackedArgs a)
{
    using namespace tc;
    using Sh = Shape<HD>;
    constexpr int ST = Sh::STAGES;
    using Bx = Bars<ST>;
    constexpr uint32_t IDESC_S = idesc_f16<T>(128, KH);
    constexpr uint32_t IDESC_O = idesc_f16<T>(128, HD) | (1u << 16);  // values read N-major
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* q_s = smem;                    // tile x at x * TILE
    unsigned char* k_s = q_s + 2 * Sh::TILE;      // stage s at s * TILE
    unsigned char* v_s = k_s + ST * Sh::TILE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + ST * Sh::TILE);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + Bx::N);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const uint32_t ny = a.kv_heads * a.nchunk, y = blockIdx.x % ny;
    PackedArgs pair = a;  // a CTA has two tiles of a.tpt tokens
    pair.tpt = 2 * a.tpt;
    const PackedTile p = packed_tile<THREADS>(pair, blockIdx.x / ny);
    if (!p.live) return;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t kvh = y / a.nchunk, hc = (y % a.nchunk) * a.gs;
    const uint32_t nh = min(a.gs, a.group - hc);                        // query heads of the tiles
    const uint32_t tokens = min(pair.tpt, p.lq - p.t0);
    const uint32_t tok0 = min(a.tpt, tokens), tok1 = tokens - tok0;     // tokens of tile A, B
    // halves of tile A and B, and the key tiles that hold them
    const uint32_t n0 = (keys_seen(p, p.t0 + tok0 - 1) + KH - 1) / KH;
    const uint32_t n1 = tok1 ? (keys_seen(p, p.t0 + tokens - 1) + KH - 1) / KH : 0u;
    const uint32_t nt0 = (n0 + 1) / 2, nt1 = (n1 + 1) / 2, ntiles = max(nt0, nt1);
    // keys of the last tile that are the sequence's
    const uint32_t tail = ntiles ? min((uint32_t)KT, p.lk - (ntiles - 1) * KT) : (uint32_t)KT;

    if (tid == 0)
    {
        for (int i = 0; i < Bx::N; ++i)
            mbar_init(&bars[i], i == B_VR ? 32u : i >= B_P0 && i < B_P0 + 4 ? 128u : 1u);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    // Registers: launched with 384 x 168; a softmax thread holds a row of 128
    // scores (2 x 128 x 208 + 128 x 80 fit the launch's)
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    if (warp < 8)
    {
        // ---------------- softmax of tile x ----------------
        const int x = warp >> 2;
        const uint32_t n = x ? n1 : n0;
        const uint32_t r = 32 * (warp & 3) + lane, tok = r / a.gs, head = r % a.gs;
        const bool live = tok < (x ? tok1 : tok0) && head < nh;
        const uint32_t token = p.t0 + (x ? a.tpt : 0u) + tok;
        // keys the row sees; rows that are no query's are left unmasked
        const uint32_t seen = live ? keys_seen(p, token) : 0xffffffffu;
        const uint32_t least = __reduce_min_sync(FULL_MASK, seen);
        const uint32_t tx = tmem + Sh::TX * x + ((uint32_t)(32 * (warp & 3)) << 16);
        // P is 2^(s - m + LIFT), at most 2^(RISE + LIFT): bf16 has fp32's range
        constexpr float LIFT = std::is_same_v<T, __half> ? 7.f : 0.f, RISE = std::is_same_v<T, __half> ? 8.f : 40.f;
        const float sl2 = a.scale * 1.4426950408889634f;  // scores in log2 units; scale > 0
        float m = -INFINITY;  // running maximum, in log2 units
        float2 l2 = make_float2(0.f, 0.f);
        bool ok = true;
        for (uint32_t i = 0; i < n; ++i)
        {
            ok = __all_sync(FULL_MASK, mbar_wait_or(&bars[B_S0 + 2 * x + (i & 1u)], i >> 1, abort));
            if (!ok) break;
            tc_fence_after();
            const uint32_t k0 = i * KH, ts = tx + KH * (i & 1u);
            const bool masked = k0 + KH > least;  // the same in the whole warp
            const int reach = (int)min(seen - k0, (uint32_t)KH) * (seen > k0);  // keys of this half that the row sees
            // P against the maximum so far; where a row's maximum has risen too
            // far, its output is rescaled and P computed again (as is the first)
            uint32_t w[32];
            float2 sum;
            while (true)
            {
                const float base = m == -INFINITY ? 0.f : LIFT - m;  // no key yet: 2^(-inf) = 0
                const float2 scale2 = make_float2(sl2, sl2), base2 = make_float2(base, base);
                uint32_t u[2][32];
                tmem_ld32_async(ts, u[0]);
                tmem_ld32_async(ts + 32, u[1]);
                sum = make_float2(0.f, 0.f);
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tmem_wait_ld(u[0]);
                tmem_wait_ld(u[1]);
#pragma unroll
                for (int c = 0; c < 2; ++c)
                {
                    mask32(u[c], masked, reach - 32 * c);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                    {
                        const float s0 = __uint_as_float(u[c][2 * j]), s1 = __uint_as_float(u[c][2 * j + 1]);
                        mx[j & 3] = max3(mx[j & 3], s0, s1);
                        const float2 e = fma2(make_float2(s0, s1), scale2, base2);
                        const float2 q = make_float2(ex2_approx(e.x), ex2_approx(e.y));
                        sum = add2(sum, q);
                        w[16 * c + j] = pack2<T>(q.x, q.y);
                    }
                }
                const float mt = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * sl2;
                const bool need = mt > m + RISE;
                if (!__any_sync(FULL_MASK, need)) break;
                const float mn = need ? mt : m;
                const float corr = need ? ex2_approx(m - mn) : 1.0f;
                l2.x *= corr;
                l2.y *= corr;
                m = mn;
                if (i > 0)
                {
                    // the product of half i - 1 must have gone into the output
                    // (that of i - 2 has: S of half i was issued after it)
                    if (!(ok = __all_sync(FULL_MASK, mbar_wait_or(&bars[B_O0 + x], i - 1, abort)))) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < HD; c += 32)
                    {
                        float v[32];
                        uint32_t o[32];
                        tmem_ld32(tx + Sh::O + c, v);
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(v[j] * corr);
                        tmem_st32(tx + Sh::O + c, o);
                    }
                }
            }
            if (!ok) break;
            l2 = add2(l2, sum);
            tmem_st32(ts, w);  // over scores that have been read
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars[B_P0 + 2 * x + (i & 1u)]);
        }
        if (ok && n > 0)
        {
            // every product of the tile is done (a barrier of one phase: this
            // thread has not followed the output's, and may be two behind)
            ok = __all_sync(FULL_MASK, mbar_wait_or(&bars[B_FIN + x], 0, abort));
            tc_fence_after();
        }
        if (ok)
        {
            const float l = l2.x + l2.y, inv = l == 0.f ? 0.f : 1.0f / l;
            T* dst = out + (uint64_t)(p.q0 + token) * a.ldo + (uint64_t)(kvh * a.group + hc + head) * HD;
            if (n == 0)
            {
                if (live)
                    for (int c = 0; c < HD; c += 8) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
            }
            else
#pragma unroll
                for (int c = 0; c < HD; c += 32)
                {
                    float v[32];
                    tmem_ld32(tx + Sh::O + c, v);
                    if (live)
#pragma unroll
                        for (int i = 0; i < 32; i += 8)
                            *reinterpret_cast<uint4*>(dst + c + i) =
                                seen ? make_uint4(pack2<T>(v[i] * inv, v[i + 1] * inv), pack2<T>(v[i + 2] * inv, v[i + 3] * inv),
                                                  pack2<T>(v[i + 4] * inv, v[i + 5] * inv), pack2<T>(v[i + 6] * inv, v[i + 7] * inv))
                                     : make_uint4(0u, 0u, 0u, 0u);
                }
        }
    }
    else if (warp < 10)
    {
        // ---------------- MMA issue for tile x ----------------
        const int x = warp - 8;
        const uint32_t n = x ? n1 : n0;
        if (n > 0)
        {
            auto wait = [&](int b, uint32_t ph) { return __all_sync(FULL_MASK, mbar_wait_or(&bars[b], ph, abort)); };
            const uint64_t dq = Sh::KDESC | (uint64_t)(smem_u32(q_s + x * Sh::TILE) >> 4);
            const uint64_t dk = Sh::KDESC | (uint64_t)(smem_u32(k_s) >> 4);
            const uint64_t dv = Sh::VDESC | (uint64_t)(smem_u32(v_s) >> 4);
            const uint32_t ts = tmem + Sh::TX * x, to = ts + Sh::O;
            // S of half i into its buffer; the last half of a key tile frees it
            auto scores = [&](uint32_t i) {
                const uint32_t st = (i >> 1) % ST, buf = i & 1u;
                const uint64_t kb = dk + ((st * Sh::TILE + buf * KH * Sh::ROW) >> 4);
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < Sh::BOXES; ++j)
#pragma unroll
                    for (int kk = 0; kk < Sh::COLS / 16; ++kk)
                    {
                        const uint32_t off = (j * Sh::BOX + kk * 32) >> 4;
                        mma_f16_ss(ts + KH * buf, dq + off, kb + off, IDESC_S, j > 0 || kk > 0);
                    }
                commit(&bars[B_S0 + 2 * x + buf]);
                if (buf || i + 1 == n) commit(&bars[Bx::KE + ST * x + st]);
            };
            bool ok = wait(B_QF, 0) && wait(Bx::KF, 0);
            if (ok) scores(0);
            if (ok && n > 1) scores(1);
            for (uint32_t i = 0; ok && i < n; ++i)
            {
                const uint32_t t = i >> 1, st = t % ST, buf = i & 1u;
                if (!buf)
                {
                    if (!(ok = wait(Bx::VF + st, t / ST))) break;
                    if (t == ntiles - 1 && tail < KT && !(ok = wait(B_VR, 0))) break;
                }
                // O += P V of half i
                if (!(ok = wait(B_P0 + 2 * x + buf, t))) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < KH / 16; ++kk)
                    mma_f16_ts(to, ts + KH * buf + 8 * kk, dv + ((st * Sh::TILE + (buf * KH + kk * 16) * Sh::ROW) >> 4),
                               IDESC_O, i > 0 || kk > 0);
                commit(&bars[B_O0 + x]);
                if (buf || i + 1 == n) commit(&bars[Bx::VE + ST * x + st]);
                if (i + 2 < n)
                {
                    // S of half i + 2, once P of half i, in the same buffer, has been read
                    if (!buf && !(ok = wait(Bx::KF + (t + 1) % ST, (t + 1) / ST))) break;
                    if (!(ok = wait(B_O0 + x, i))) break;
                    scores(i + 2);
                }
            }
            // every MMA this warp issued completes before TMEM is freed
            commit(&bars[B_FIN + x]);
            __all_sync(FULL_MASK, mbar_wait(&bars[B_FIN + x], 0));
        }
    }
    else if (warp == 10)
    {
        // ---------------- TMA copies ----------------
        uint32_t last = 0;  // copies issued
        if (lane == 0 && ntiles > 0)
        {
            const uint32_t nq = nt1 ? 2u : 1u;
            mbar_arrive_expect_tx(&bars[B_QF], nq * Sh::BOXES * a.gs * a.tpt * Sh::ROW);
            for (uint32_t x = 0; x < nq; ++x)
                for (int j = 0; j < Sh::BOXES; ++j)
                    tma_load_3d(q_s + x * Sh::TILE + j * Sh::BOX, &map_q, Sh::COLS * j, (int)(kvh * a.group + hc),
                                (int)(p.q0 + p.t0 + x * a.tpt), &bars[B_QF]);
            uint32_t issued = 0;  // copies: K(t) is 2 t, V(t) is 2 t + 1
            for (uint32_t t = 0; t < ntiles; ++t)
            {
                const uint32_t st = t % ST, ph = t / ST;
                // into stage st once both query tiles' products have read what it held
                auto freed = [&](int e) {
                    return t < (uint32_t)ST || ((t - ST >= nt0 || mbar_wait_or(&bars[e + st], ph - 1, abort)) &&
                                                (t - ST >= nt1 || mbar_wait_or(&bars[e + ST + st], ph - 1, abort)));
                };
                if (!freed(Bx::KE)) break;
                mbar_arrive_expect_tx(&bars[Bx::KF + st], Sh::TILE);
                for (int j = 0; j < Sh::BOXES; ++j)
                    tma_load_2d(k_s + st * Sh::TILE + j * Sh::BOX, &map_k, (int)(kvh * HD) + Sh::COLS * j,
                                (int)(p.k0 + t * KT), &bars[Bx::KF + st]);
                issued = 2 * t + 1;
                if (!freed(Bx::VE)) break;
                mbar_arrive_expect_tx(&bars[Bx::VF + st], Sh::TILE);
                for (int j = 0; j < Sh::BOXES; ++j)
                    tma_load_2d(v_s + st * Sh::TILE + j * Sh::BOX, &map_v, (int)(kvh * HD) + Sh::COLS * j,
                                (int)(p.k0 + t * KT), &bars[Bx::VF + st]);
                issued = 2 * t + 2;
            }
            last = issued;
        }
        // Rows past the sequence's end in its last value tile.  The copy loop
        // has seen every earlier phase of the stage's barrier complete.
        __syncwarp();
        last = __shfl_sync(FULL_MASK, last, 0);
        if (tail < KT && ntiles > 0 && last == 2 * ntiles)
        {
            const uint32_t st = (ntiles - 1) % ST;
            if (mbar_wait_or(&bars[Bx::VF + st], (ntiles - 1) / ST, abort))
            {
                for (int j = 0; j < Sh::BOXES; ++j)
                {
                    uint4* box = reinterpret_cast<uint4*>(v_s + st * Sh::TILE + j * Sh::BOX);
                    for (uint32_t i = tail * (Sh::ROW / 16) + lane; i < Sh::BOX / 16; i += 32)
                        box[i] = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_async_smem();
                mbar_arrive(&bars[B_VR]);
            }
        }
        if (lane == 0 && ntiles > 0)
        {
            // the copies this thread started land before the CTA exits (bounded)
            mbar_wait(&bars[B_QF], 0);
            for (uint32_t n = last > 2 * ST ? last - 2 * ST : 0; n < last; ++n)
            {
                const uint32_t t = n >> 1;
                mbar_wait(&bars[(n & 1u ? Bx::VF : Bx::KF) + t % ST], (t / ST) & 1u);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort) atomicAdd(&g_packed_tc_timeouts, 1);
    if (warp == 0)
    {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

namespace {

// [rows][heads][cols] 16-bit elements (row stride ld) as boxes of `box_cols` x
// box_heads x box_rows; what lies outside reads as zero.
int make_map_16(CUtensorMap* map, const void* base, int type, uint32_t cols, uint32_t heads, uint32_t rows, uint32_t ld,
                uint32_t box_cols, uint32_t box_heads, uint32_t box_rows, bool flat)
{
    auto enc = tc::get_encode();
    if (!enc) return set_error(FML_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    // flat: [rows][heads * cols]
    const cuuint64_t dims[3] = {flat ? (cuuint64_t)cols * heads : cols, flat ? rows : heads, rows};
    const cuuint64_t strides[2] = {flat ? (cuuint64_t)ld * 2 : (cuuint64_t)cols * 2, (cuuint64_t)ld * 2};
    const cuuint32_t box[3] = {box_cols, flat ? box_rows : box_heads, box_rows};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, type == FML_TYPE_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           flat ? 2 : 3, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(FML_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FML_OK;
}

template <typename T, int HD>
int launch(void* out, const void* q, const void* k, const void* v, int type, PackedArgs a, cudaStream_t st)
{
    using Sh = Shape<HD>;
    auto kern = packed_attention_tc_kernel<T, HD>;
    static uint64_t attr_devices = 0;
    FML_RC(smem_limit_once(reinterpret_cast<const void*>(kern), (int)Sh::SMEM, attr_devices));
    a.gs = a.group < 128u ? a.group : 128u;
    a.nchunk = (a.group + a.gs - 1) / a.gs;
    a.tpt = 128u / a.gs;
    PackedArgs pair = a;
    pair.tpt = 2 * a.tpt;
    const uint64_t ctas = packed_tiles_bound(pair) * a.kv_heads * a.nchunk;
    FML_REQUIRE(ctas < (1ull << 31), "fml_attention_packed: %u rows of %u heads", a.q_rows, a.heads);
    CUtensorMap mq, mk, mv;
    FML_RC(make_map_16(&mq, q, type, HD, a.heads, a.q_rows, a.ldq, Sh::COLS, a.gs, a.tpt, false));
    FML_RC(make_map_16(&mk, k, type, HD, a.kv_heads, a.k_rows, a.ldk, Sh::COLS, 1, KT, true));
    FML_RC(make_map_16(&mv, v, type, HD, a.kv_heads, a.k_rows, a.ldv, Sh::COLS, 1, KT, true));
    kern<<<(unsigned)ctas, THREADS, Sh::SMEM, st>>>(mq, mk, mv, static_cast<T*>(out), a);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

}  // namespace

// The tensor-core kernel for 16-bit inputs; FML_ERR_UNSUPPORTED (no error
// recorded) for what it does not take: bases and row strides that are not
// multiples of 16 bytes (TMA's rule), a scale that is not positive (the
// maximum is taken before the scale), or no key row at all.
int launch_packed_attention_tc(void* out, const void* q, const void* k, const void* v, int type, uint32_t head_dim,
                               const PackedArgs& a, cudaStream_t st)
{
    if (!(a.scale > 0.f) || a.k_rows == 0 || !aligned16(out) || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
        (a.ldo | a.ldq | a.ldk | a.ldv) % 8)
        return FML_ERR_UNSUPPORTED;
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (head_dim == 32) return launch<T, 32>(out, q, k, v, type, a, st);
        if (head_dim == 64) return launch<T, 64>(out, q, k, v, type, a, st);
        return launch<T, 128>(out, q, k, v, type, a, st);
    };
    if (type == FML_TYPE_FP16) return go(static_cast<__half*>(nullptr));
    return go(static_cast<__nv_bfloat16*>(nullptr));
}

int packed_tc_error_count(int* out)
{
    FML_CUDA_TRY(cudaMemcpyFromSymbol(out, g_packed_tc_timeouts, sizeof(int)));
    return FML_OK;
}

}  // namespace fml
