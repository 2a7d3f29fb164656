// Causal attention over packed prompts with grouped heads, fp16 and bf16, on
// the tensor cores: S = Q K^T * scale with the causal mask, row softmax, P V,
// as one pass over the keys with a running maximum and sum.
//
// A CTA stays on its SM and takes one work item after another, the heaviest
// first: two tiles, A and B, of 128 query rows of one key/value head (packed.cuh: tokens in order and,
// for each, the query heads of the group, so that a group shares every key and
// value tile).  The grid has a block for every item; a running CTA takes over
// blocks that have not started (cluster launch control), so that items of very
// different lengths even out and barriers, TMEM and registers are set up once.
//   warps 0-3, 4-7  softmax of tile A, B (thread = TMEM lane = query row)
//   warps 8, 9      issue tile A's / B's S products (tcgen05.mma, one lane elected)
//   warps 10, 11    issue their P V products
//   warp 12         issues every TMA copy and zeroes the rows past the
//                   sequence's end in its last value tile (another sequence's
//                   rows, or its NaN, lie there)
//   warp 13         finds the next item (14 and 15 are idle: registers are
//                   shared out by groups of four warps)
// Each role runs ahead into the next item as far as its barriers let it: its
// queries are copied while the last products of this one run, its first scores
// are there when the softmax warps have written this one's output.
// Keys and values are copied 128 rows at a time and used in halves of 64.  TMEM,
// per query tile: two score buffers of 64 fp32 columns, S of half i in buffer
// i % 2, overwritten in place by P in 16 bits (32 columns, the A operand of
// O += P V, read from TMEM), and the output's hd columns, which stay there over
// all keys.  With two buffers S of half i + 1 is there before P of half i is, and
// the softmax warps never wait for a product in the steady state (one buffer of
// 128 keys, whose S product costs the tensor cores less, was slower: S, softmax
// and P V then follow one another).
// A row rescales its output only when a score rises by more than 2^8 (bf16:
// 2^40) over the maximum that its P is taken against; fp16 P is taken 2^7
// larger, so that it uses the type's range (at most 2^15) and small
// probabilities stay above its smallest numbers.
//
// What bounds it: a half of 64 keys of both tiles takes about 2050 cycles in head
// dim 128, of which the tensor cores work 1280 (S of 64 keys takes 3/4 of the
// time of one of 128: shared memory's rate) and the special function units 1024.
// The softmax warps, one of each tile to a scheduler, are what the rest waits
// for: wait, ld, maximum, exponentials and st follow one another.  Tried and not
// faster: four softmax warps a scheduler (a half's latency then bounds the two
// buffers), turns at the exponentials, polynomials for a part of them.
// Grouped bf16 prompts of up to 4096 (2.1e11 flops, head dim 128) take 257 us,
// 0.82 PFLOP/s; fp16 ones of up to 1537, 16 heads of 64 (3.5e10), 124 us.
// P in 16 bits costs, in the norm, at most as much as the result's own rounding
// (fp16 2.0e-4 -> 2.4e-4, bf16 1.6e-3 -> 2.0e-3 on these cases, about sqrt(2) times at the most).
// As two halves it would fit the score buffer, but double the P V products and add
// two conversions a score to the warps that the rest waits for.
// O stays in TMEM over all keys, where the tensor cores cut their running sums: of
// values whose mean is not 0, fp16 outputs are 2.7e-4 off behind 32,000 keys (plain
// 2.2e-4) and 6.4e-4 behind 128,000; bf16 ones 1.87e-3, for a rounding of 1.79e-3.
// Every wait is bounded and returns early once any role has recorded an expiry.
// A wait tells neighbouring phases of a barrier apart only, so every role that
// waits on a barrier follows all of its phases, or is never two behind.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>
#include <cuda/ptx>

#include "f32x2.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace fml {

__device__ int g_packed_tc_timeouts;

namespace {

constexpr int THREADS = 16 * 32;
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
    static constexpr uint32_t SMEM = 2 * TILE + 2 * STAGES * TILE + 1024 + 1024 + 8 * 2048;
    // TMEM columns of tile x: S / P buffers 0 and 1, the output
    static constexpr uint32_t TX = 256, O = 2 * KH;
    // shared-memory operand descriptors: 8-row groups of the swizzled rows
    static constexpr uint64_t LAYOUT = HD < 64 ? 4ull << 61 : 2ull << 61;  // 64- or 128-byte swizzle
    static constexpr uint64_t SBO = (uint64_t)(8 * ROW >> 4) << 32;
    static constexpr uint64_t KDESC = LAYOUT | SBO | (1ull << 16) | (1ull << 46);
    // value tile as an N-major operand: the next columns a box on, the next 8 keys a row group on
    static constexpr uint64_t VDESC = LAYOUT | SBO | ((uint64_t)(BOX >> 4) << 16) | (1ull << 46);
};

// Items: found and taken (two slots), queries landed and consumed, the launch
// control's answer.  Per query tile x: S, P and P V by buffer (2 x + buffer), the
// item's output done and read, the end of both issuing warps.  Per stage: K and V
// copies landed, rows past a sequence's end zeroed, K and V consumed by both
// query tiles.
enum Bar { B_TF, B_TE = B_TF + 2, B_QF = B_TE + 2, B_QE, B_CL, B_S0, B_P0 = B_S0 + 4, B_O0 = B_P0 + 4,
           B_OD = B_O0 + 4, B_OE = B_OD + 2, B_FIN = B_OE + 2, B_KF = B_FIN + 4 };
template <int ST>
struct Bars
{
    static constexpr int KF = B_KF, VF = KF + ST, VR = VF + ST, KE = VR + ST, VE = KE + ST, N = VE + ST;
    __device__ static constexpr uint32_t arrivals(int i)
    {
        if (i == B_TE || i == B_TE + 1) return 13;  // 8 softmax, 4 MMA warps, the copying one
        if (i == B_QE || (i >= KE && i < N)) return 2;  // both query tiles' MMA warps
        if (i >= VR && i < KE) return 32;
        if ((i >= B_P0 && i < B_P0 + 4) || i == B_OE || i == B_OE + 1) return 128;
        return 1;
    }
};

// A work item, as the finder leaves it for the others.
struct Item
{
    PackedTile p;        // live 0: no more
    uint32_t kvh, hc;    // key/value head, first query head of the group
    uint32_t tok0, tok1; // tokens of tile A, B
    uint32_t n0, n1;     // halves of their keys
    uint32_t ntiles;     // key tiles that hold them
    uint32_t tail;       // keys of the last tile that are the sequence's
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

// A value that is the same in the whole warp, as the compiler cannot see: an
// operand of it then needs no loop over the lanes' values.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __shfl_sync(FULL_MASK, x, 0); }

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
    uint4* answer = reinterpret_cast<uint4*>(bars + (Bx::N + 1) / 2 * 2);  // of the launch control
    Item* items = reinterpret_cast<Item*>(answer + 1);                    // two slots
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(items + 2);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint4* staging = reinterpret_cast<uint4*>(v_s + ST * Sh::TILE + 1024);  // 2 KB a softmax warp
    static_assert((Bx::N + 1) / 2 * 16 + 16 + 2 * sizeof(Item) + 8 <= 1024, "the barriers' room");

    const int tid = threadIdx.x, warp = (int)uniform(tid >> 5), lane = tid & 31;
    if (tid == 0)
    {
        for (int i = 0; i < Bx::N; ++i) mbar_init(&bars[i], Bx::arrivals(i));
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
    const uint32_t tmem = uniform(*tmem_slot);
    // a bounded wait of the whole warp
    auto wait = [&](int b, uint32_t ph) { return __all_sync(FULL_MASK, mbar_wait_or(&bars[b], ph, abort)) != 0; };
    // item k, once it is there (false: a wait has expired); its slot given back
    auto take = [&](uint32_t k, Item* it) {
        if (!wait(B_TF + (k & 1u), k >> 1)) return false;
        *it = items[k & 1u];
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[B_TE + (k & 1u)]);
        return it->p.live != 0;
    };

    // Registers: launched with 512 x 128, shared out as 2 x 128 x 192 for the
    // softmax warps and 2 x 128 x 64
    if (warp < 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp < 8)
    {
        // ---------------- softmax of tile x ----------------
        const int x = warp >> 2;
        const uint32_t r = 32 * (warp & 3) + lane, tok = r / a.gs, head = r % a.gs;
        const uint32_t tx = tmem + Sh::TX * x + ((uint32_t)(32 * (warp & 3)) << 16);
        // P is 2^(s - m + LIFT), at most 2^(RISE + LIFT): bf16 has fp32's range
        constexpr float LIFT = std::is_same_v<T, __half> ? 7.f : 0.f, RISE = std::is_same_v<T, __half> ? 8.f : 40.f;
        const float sl2 = a.scale * 1.4426950408889634f;  // scores in log2 units; scale > 0
        uint32_t g = 0, done = 0;  // halves and items of this tile so far
        Item it;
        for (uint32_t k = 0; take(k, &it); ++k)
        {
            const uint32_t n = x ? it.n1 : it.n0;
            const bool live = tok < (x ? it.tok1 : it.tok0) && head < min(a.gs, a.group - it.hc);
            const uint32_t token = it.p.t0 + (x ? a.tpt : 0u) + tok;
            // keys the row sees; rows that are no query's are left unmasked
            const uint32_t seen = live ? keys_seen(it.p, token) : 0xffffffffu;
            const uint32_t least = __reduce_min_sync(FULL_MASK, seen);
            float m = -INFINITY;  // the row's reference, in log2 units
            float2 l2 = make_float2(0.f, 0.f);
            bool ok = true;
            for (uint32_t i = 0; i < n; ++i, ++g)
            {
                if (!(ok = wait(B_S0 + 2 * x + (g & 1u), g >> 1))) break;
                tc_fence_after();
                const uint32_t k0 = i * KH, ts = tx + KH * (g & 1u);
                const bool masked = k0 + KH > least;  // the same in the whole warp
                const int reach = (int)min(seen - k0, (uint32_t)KH) * (seen > k0);  // keys of this half that the row sees
                // P against the reference; where a score has risen too far over
                // it, the output is rescaled and P computed again (as is the first)
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
                        // the product of the half before must have gone into the
                        // output (the one before it has: S was issued after it)
                        if (!(ok = wait(B_O0 + 2 * x + ((g - 1) & 1u), (g - 1) >> 1))) break;
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
                mbar_arrive(&bars[B_P0 + 2 * x + (g & 1u)]);
            }
            if (!ok) break;
            // The output, 32 columns at a time through shared memory: rows lie
            // far apart, and a store of 16 bytes of each of 32 rows costs the
            // memory unit 32 steps, one of 64 bytes of 8 rows 8.
            const float l = l2.x + l2.y, inv = l == 0.f ? 0.f : 1.0f / l;
            if (n > 0 && !wait(B_OD + x, done++)) break;
            tc_fence_after();
            const uint64_t row = (uint64_t)(it.p.q0 + token) * a.ldo + (uint64_t)(it.kvh * a.group + it.hc + head) * HD;
            uint4* stage = staging + warp * 128;  // 32 rows of 4 x 16 bytes, chunk j of row i at j ^ (i >> 1 & 3)
#pragma unroll
            for (int c = 0; c < HD; c += 32)
            {
                float v[32];
                if (n > 0)
                {
                    tmem_ld32(tx + Sh::O + c, v);
                    if (c + 32 == HD)
                    {
                        tc_fence_before();
                        mbar_arrive(&bars[B_OE + x]);  // the next item's products may overwrite the output
                    }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const uint4 q = make_uint4(pack2<T>(v[8 * j] * inv, v[8 * j + 1] * inv), pack2<T>(v[8 * j + 2] * inv, v[8 * j + 3] * inv),
                                               pack2<T>(v[8 * j + 4] * inv, v[8 * j + 5] * inv), pack2<T>(v[8 * j + 6] * inv, v[8 * j + 7] * inv));
                    stage[4 * lane + (j ^ (lane >> 1 & 3))] = n > 0 && seen ? q : make_uint4(0u, 0u, 0u, 0u);
                }
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    const int i = 8 * j + (lane >> 2);  // row of the warp; 4 lanes each
                    const uint64_t at = __shfl_sync(FULL_MASK, row, i);
                    const bool there = __shfl_sync(FULL_MASK, (int)live, i);
                    const uint4 q = stage[4 * i + ((lane & 3) ^ (i >> 1 & 3))];
                    if (there) *reinterpret_cast<uint4*>(out + at + c + 8 * (lane & 3)) = q;
                }
                __syncwarp();
            }
        }
    }
    else if (warp < 10)
    {
        // ---------------- S of tile x ----------------
        const int x = warp - 8;
        const uint64_t dq = Sh::KDESC | (uint64_t)(smem_u32(q_s + x * Sh::TILE) >> 4);
        const uint64_t dk = Sh::KDESC | (uint64_t)(smem_u32(k_s) >> 4);
        const uint32_t ts = tmem + Sh::TX * x;
        uint32_t g = 0, tiles = 0, queries = 0;  // halves, key tiles and items so far
        bool ok = true;
        Item it;
        for (uint32_t k = 0; ok && take(k, &it); ++k)
        {
            if (it.ntiles == 0) continue;
            const uint32_t n = uniform(x ? it.n1 : it.n0), ntiles = uniform(it.ntiles);
            if (!(ok = wait(B_QF, queries++))) break;
            for (uint32_t t = 0; ok && t < ntiles; ++t, ++tiles)
            {
                const uint32_t st = tiles % ST;
                if (!(ok = wait(Bx::KF + st, tiles / ST))) break;
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half)
                    if (2 * t + half < n)
                    {
                        // its buffer: P V of the half before last has read it
                        if (g >= 2 && !(ok = wait(B_O0 + 2 * x + (g & 1u), (g >> 1) - 1))) break;
                        const uint64_t kb = dk + ((st * Sh::TILE + half * KH * Sh::ROW) >> 4);
                        tc_fence_after();
#pragma unroll
                        for (int j = 0; j < Sh::BOXES; ++j)
#pragma unroll
                            for (int kk = 0; kk < Sh::COLS / 16; ++kk)
                            {
                                const uint32_t off = (j * Sh::BOX + kk * 32) >> 4;
                                mma_f16_ss(ts + KH * (g & 1u), dq + off, kb + off, IDESC_S, j > 0 || kk > 0);
                            }
                        commit(&bars[B_S0 + 2 * x + (g & 1u)]);
                        ++g;
                    }
                if (!ok) break;
                commit(&bars[Bx::KE + st]);  // a tile is given back, used or not
            }
            if (ok) commit(&bars[B_QE]);
        }
        // every MMA this warp issued completes before TMEM is freed
        commit(&bars[B_FIN + x]);
        __all_sync(FULL_MASK, mbar_wait(&bars[B_FIN + x], 0));
    }
    else if (warp < 12)
    {
        // ---------------- P V of tile x ----------------
        const int x = warp - 10;
        const uint64_t dv = Sh::VDESC | (uint64_t)(smem_u32(v_s) >> 4);
        const uint32_t ts = tmem + Sh::TX * x, to = ts + Sh::O;
        // halves, key tiles and items of this query tile so far; by stage, zeroed tiles' parity
        uint32_t g = 0, tiles = 0, outputs = 0, ends = 0;
        bool ok = true;
        Item it;
        for (uint32_t k = 0; ok && take(k, &it); ++k)
        {
            if (it.ntiles == 0) continue;
            const uint32_t n = uniform(x ? it.n1 : it.n0), ntiles = uniform(it.ntiles), tail = uniform(it.tail);
            for (uint32_t t = 0; ok && t < ntiles; ++t, ++tiles)
            {
                const uint32_t st = tiles % ST;
                if (!(ok = wait(Bx::VF + st, tiles / ST))) break;
                if (t + 1 == ntiles && tail < KT)
                {
                    if (!(ok = wait(Bx::VR + st, ends >> st & 1u))) break;
                    ends ^= 1u << st;
                }
#pragma unroll
                for (uint32_t half = 0; half < 2; ++half)
                    if (2 * t + half < n)
                    {
                        // the item's first overwrites an output that has been read
                        if (t == 0 && half == 0 && outputs > 0 && !(ok = wait(B_OE + x, outputs - 1))) break;
                        if (!(ok = wait(B_P0 + 2 * x + (g & 1u), g >> 1))) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < KH / 16; ++kk)
                            mma_f16_ts(to, ts + KH * (g & 1u) + 8 * kk,
                                       dv + ((st * Sh::TILE + (half * KH + kk * 16) * Sh::ROW) >> 4), IDESC_O,
                                       t > 0 || half > 0 || kk > 0);
                        commit(&bars[B_O0 + 2 * x + (g & 1u)]);
                        if (2 * t + half + 1 == n) commit(&bars[B_OD + x]);
                        ++g;
                    }
                if (!ok) break;
                commit(&bars[Bx::VE + st]);
            }
            outputs += n > 0;
        }
        commit(&bars[B_FIN + 2 + x]);
        __all_sync(FULL_MASK, mbar_wait(&bars[B_FIN + 2 + x], 0));
    }
    else if (warp == 12)
    {
        // ---------------- TMA copies ----------------
        uint32_t tiles = 0, queries = 0;  // so far
        uint32_t kcopies = 0, vcopies = 0, qcopies = 0;
        Item it;
        for (uint32_t k = 0; take(k, &it); ++k)
        {
            if (it.ntiles == 0) continue;
            if (queries > 0 && !wait(B_QE, queries - 1)) break;
            if (lane == 0)
            {
                const uint32_t nq = it.tok1 ? 2u : 1u;
                mbar_arrive_expect_tx(&bars[B_QF], nq * Sh::BOXES * a.gs * a.tpt * Sh::ROW);
                for (uint32_t x = 0; x < nq; ++x)
                    for (int j = 0; j < Sh::BOXES; ++j)
                        tma_load_3d(q_s + x * Sh::TILE + j * Sh::BOX, &map_q, Sh::COLS * j, (int)(it.kvh * a.group + it.hc),
                                    (int)(it.p.q0 + it.p.t0 + x * a.tpt), &bars[B_QF]);
            }
            ++qcopies;
            bool ok = true;
            for (uint32_t t = 0; t < it.ntiles; ++t)
            {
                const uint32_t tile = tiles + t, st = tile % ST, ph = tile / ST;
                // into stage st once both query tiles' products have read what it held
                if (ph > 0 && !(ok = wait(Bx::KE + st, ph - 1))) break;
                if (lane == 0)
                {
                    mbar_arrive_expect_tx(&bars[Bx::KF + st], Sh::TILE);
                    for (int j = 0; j < Sh::BOXES; ++j)
                        tma_load_2d(k_s + st * Sh::TILE + j * Sh::BOX, &map_k, (int)(it.kvh * HD) + Sh::COLS * j,
                                    (int)(it.p.k0 + t * KT), &bars[Bx::KF + st]);
                }
                ++kcopies;
                if (ph > 0 && !(ok = wait(Bx::VE + st, ph - 1))) break;
                if (lane == 0)
                {
                    mbar_arrive_expect_tx(&bars[Bx::VF + st], Sh::TILE);
                    for (int j = 0; j < Sh::BOXES; ++j)
                        tma_load_2d(v_s + st * Sh::TILE + j * Sh::BOX, &map_v, (int)(it.kvh * HD) + Sh::COLS * j,
                                    (int)(it.p.k0 + t * KT), &bars[Bx::VF + st]);
                }
                ++vcopies;
                if (t + 1 == it.ntiles && it.tail < KT)
                {
                    // rows past the sequence's end
                    if (!(ok = wait(Bx::VF + st, ph))) break;
                    for (int j = 0; j < Sh::BOXES; ++j)
                    {
                        uint4* box = reinterpret_cast<uint4*>(v_s + st * Sh::TILE + j * Sh::BOX);
                        for (uint32_t i = it.tail * (Sh::ROW / 16) + lane; i < Sh::BOX / 16; i += 32)
                            box[i] = make_uint4(0u, 0u, 0u, 0u);
                    }
                    fence_async_smem();
                    mbar_arrive(&bars[Bx::VR + st]);
                }
            }
            if (!ok) break;
            tiles += it.ntiles;
            ++queries;
        }
        // the copies this warp started land before the CTA exits (bounded)
        if (qcopies > 0) mbar_wait(&bars[B_QF], (qcopies - 1) & 1u);
        for (uint32_t i = kcopies > ST ? kcopies - ST : 0; i < kcopies; ++i) mbar_wait(&bars[Bx::KF + i % ST], (i / ST) & 1u);
        for (uint32_t i = vcopies > ST ? vcopies - ST : 0; i < vcopies; ++i) mbar_wait(&bars[Bx::VF + i % ST], (i / ST) & 1u);
    }
    else if (warp == 13)
    {
        // ---------------- the next item ----------------
        const uint32_t ny = a.kv_heads * a.nchunk;
        const PackedTotals all = packed_totals(a);
        uint32_t asked = 0;
        bool more = true;
        uint32_t block = blockIdx.x;
        for (uint32_t k = 0; more;)
        {
            Item it;
            it.p = packed_tile(a, all, block / ny);
            // ask for the next block while this one is worked out
            if (lane == 0)
            {
                mbar_arrive_expect_tx(&bars[B_CL], 16);
                cuda::ptx::clusterlaunchcontrol_try_cancel(answer, &bars[B_CL]);
            }
            ++asked;
            if (it.p.live)
            {
                const uint32_t y = block % ny;
                it.kvh = y / a.nchunk;
                it.hc = (y % a.nchunk) * a.gs;
                const uint32_t tokens = min(a.step, it.p.lq - it.p.t0);
                it.tok0 = min(a.tpt, tokens);
                it.tok1 = tokens - it.tok0;
                it.n0 = (keys_seen(it.p, it.p.t0 + it.tok0 - 1) + KH - 1) / KH;
                it.n1 = it.tok1 ? (keys_seen(it.p, it.p.t0 + tokens - 1) + KH - 1) / KH : 0u;
                it.ntiles = (max(it.n0, it.n1) + 1) / 2;
                it.tail = it.ntiles ? min((uint32_t)KT, it.p.lk - (it.ntiles - 1) * KT) : (uint32_t)KT;
                if (k >= 2 && !wait(B_TE + (k & 1u), (k >> 1) - 1)) break;
                if (lane == 0)
                {
                    items[k & 1u] = it;
                    mbar_arrive(&bars[B_TF + (k & 1u)]);
                }
                ++k;
            }
            if (!wait(B_CL, asked - 1)) break;
            const uint4 got = *answer;
            more = cuda::ptx::clusterlaunchcontrol_query_cancel_is_canceled(got);
            if (more) block = (uint32_t)cuda::ptx::clusterlaunchcontrol_query_cancel_get_first_ctaid_x<int>(got);
            __syncwarp();
            fence_async_smem();  // the answer has been read before the next one is written
            if (!more)
            {
                if (k >= 2 && !wait(B_TE + (k & 1u), (k >> 1) - 1)) break;
                if (lane == 0)
                {
                    items[k & 1u].p.live = 0;
                    mbar_arrive(&bars[B_TF + (k & 1u)]);
                }
            }
        }
        // an answer still on its way lands before the CTA exits (bounded; immediate on the normal path)
        mbar_wait(&bars[B_CL], (asked - 1) & 1u);
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
    const uint64_t ctas = packed_items(&a, 128, 2);
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
