// Causal prefill attention on the tensor cores: CausalSelfAttentionLayer::
// Forward (CausalSelfAttentionLayer.h:424-499) over whole prompts -- per head
// S = Q K^T * 1/sqrt(hd) + causal mask, row softmax, Y = P V -- as a
// flash-attention loop on tcgen05 with fp32-level accuracy (TF32x3).
//
// CTA = 4 warps on (128 query rows, head, sequence); it walks the key tiles
// (KT keys) up to its last row.  Per tile:
//   1. K tile (TMA, 128-byte swizzle, K-major) -> its TF32 lo part; the first
//      warp issues S = Q K^T (Q_hi K_hi + Q_hi K_lo + Q_lo K_hi) into TMEM;
//   2. thread r (= TMEM lane r) reads query row r's KT scores with
//      tcgen05.ld, scales and masks them (keys past the row and past the
//      prompt), and updates the row's online softmax (running max m and sum
//      l); it writes the row's probabilities P (and their lo part) into
//      shared memory as the K-major A operand of the next MMA;
//   3. V tile: TMA in the 128-byte swizzle of 32-byte atoms, the layout an
//      N-major tf32 operand needs (V is stored [keys x hd], hd contiguous);
//      rows past the last valid key are zeroed (the cache may hold anything
//      there); the first warp issues O_tile = P V (TF32x3) into a second TMEM
//      accumulator;
//   4. thread r reads its O_tile row and accumulates O = O corr + O_tile in
//      registers (corr = exp(m_old - m_new)).
// At the end each valid row writes O / l.  The next tile's K and V copies
// start as soon as the MMAs that read the current ones have completed.
// Every mbarrier wait is bounded (expiries are counted in the device error
// count; the CTA then stops issuing work and still frees its TMEM).
#include <cmath>
#include <cstdlib>

#include "packed.cuh"
#include "tcgen05.cuh"

namespace fml {

__device__ int g_prefill_tc_timeouts;

namespace {

constexpr int QB = 128;  // query rows per CTA (= TMEM lanes)

struct PfArgs
{
    float* out;       // [B*P x ldo], head h at column h * HD
    uint32_t ldo;
    uint32_t B, H, P, C;
    float scale;      // 1/sqrt(hd), CausalSelfAttentionLayer.h:73-77
};

template <int HD>
struct PfShape
{
    static constexpr int KT = HD <= 64 ? 64 : 32;           // keys per tile
    static constexpr uint32_t QBYTES = HD * QB * 4;          // Q tile: HD/32 blocks of [128 x 32]
    static constexpr uint32_t KBYTES = HD * KT * 4;          // K tile: HD/32 blocks of [KT x 32]
    static constexpr uint32_t VBYTES = HD * KT * 4;          // V tile: (KT/32) x (HD/32) boxes of [32 x 32]
    static constexpr uint32_t PBYTES = KT * QB * 4;          // P tile: KT/32 blocks of [128 x 32]
    static constexpr uint32_t SMEM = 2 * (QBYTES + KBYTES + VBYTES + PBYTES) + 1024 + 64;
    static constexpr uint32_t OCOL = KT < 32 ? 32 : KT;      // TMEM column of the O accumulator
    static constexpr uint32_t TCOLS = OCOL + HD <= 128 ? 128 : 256;
};

__device__ __forceinline__ void lo_inplace(float4* dst, const float4* src, uint32_t n4, int tid)
{
    for (uint32_t i = tid; i < n4; i += 128) dst[i] = tc::tf32_lo4(src[i]);
}

__device__ __forceinline__ uint64_t desc_mn(const void* tile)
{
    // MN-major, 128-byte swizzle with 32-byte atoms: the next 32 n one 4 KB
    // box on (LBO), the next 4 k one 512-byte atom on (SBO)
    const uint64_t start = (uint64_t)(tc::smem_u32(tile) >> 4) & 0x3FFFull;
    return start | ((uint64_t)(4096 >> 4) << 16) | ((uint64_t)(512 >> 4) << 32) | (1ull << 46) | (1ull << 61);
}

}  // namespace

template <int HD, bool SPLIT3>
__global__ void __launch_bounds__(128, 1) prefill_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q,
                                                                      const __grid_constant__ CUtensorMap map_k,
                                                                      const __grid_constant__ CUtensorMap map_v,
                                                                      PfArgs a)
{
    using namespace tc;
    using Sh = PfShape<HD>;
    constexpr int KT = Sh::KT;
    constexpr uint32_t IDESC_S = idesc_tf32(128, KT);
    constexpr uint32_t IDESC_O = idesc_tf32(128, HD) | (1u << 16);  // B (V) read MN-major
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* q_s = smem;
    unsigned char* qlo_s = q_s + Sh::QBYTES;
    unsigned char* k_s = qlo_s + Sh::QBYTES;
    unsigned char* klo_s = k_s + Sh::KBYTES;
    unsigned char* v_s = klo_s + Sh::KBYTES;
    unsigned char* vlo_s = v_s + Sh::VBYTES;
    unsigned char* p_s = vlo_s + Sh::VBYTES;
    unsigned char* plo_s = p_s + Sh::PBYTES;
    // barriers: Q, K, V copies; S, O products
    uint64_t* bars = reinterpret_cast<uint64_t*>(plo_s + Sh::PBYTES);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 5);
    enum { BQ = 0, BKEY = 1, BVAL = 2, BS = 3, BO = 4 };

    const int tid = threadIdx.x, warp = tid >> 5;
    const uint32_t q0 = blockIdx.x * QB, h = blockIdx.y, b = blockIdx.z;
    const uint32_t P = a.P;
    const uint32_t nkeys = min(q0 + (uint32_t)QB, P);         // keys this CTA's rows can see
    const uint32_t ntiles = (nkeys + KT - 1) / KT;
    const int kv_row0 = (int)((b * a.H + h) * a.C);           // this (sequence, head)'s first cache row
    const uint32_t q = q0 + tid;                              // this thread's query row
    // thread 0's count of the phases it started / saw complete on each barrier
    // (the drain after an expired wait)
    uint32_t issued[5] = {0, 0, 0, 0, 0}, seen[5] = {0, 0, 0, 0, 0};

    if (tid == 0)
    {
        for (int i = 0; i < 5; ++i) mbar_init(&bars[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(Sh::TCOLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = __shfl_sync(FULL_MASK, *tmem_slot, 0);  // the same in the warp for the compiler too
    const bool warp0 = __shfl_sync(FULL_MASK, warp, 0) == 0;
    const uint32_t tmem_o = tmem + Sh::OCOL;
    const uint32_t lane_base = (uint32_t)(32 * warp) << 16;

    auto issue_k = [&](uint32_t t) {
        mbar_arrive_expect_tx(&bars[BKEY], Sh::KBYTES);
        for (int j = 0; j < HD / 32; ++j)
            tma_load_2d(k_s + j * (KT * 128), &map_k, 32 * j, kv_row0 + (int)(t * KT), &bars[BKEY]);
        ++issued[BKEY];
    };
    auto issue_v = [&](uint32_t t) {
        mbar_arrive_expect_tx(&bars[BVAL], Sh::VBYTES);
        for (int kb = 0; kb < KT / 32; ++kb)
            for (int j = 0; j < HD / 32; ++j)
                tma_load_2d(v_s + (kb * (HD / 32) + j) * 4096, &map_v, 32 * j, kv_row0 + (int)(t * KT) + 32 * kb,
                            &bars[BVAL]);
        ++issued[BVAL];
    };
    // bounded wait on phase `ph` of barrier i, the same answer in the whole warp
    auto wait = [&](int i, uint32_t ph) {
        const bool w = __all_sync(FULL_MASK, mbar_wait(&bars[i], ph & 1u));
        if (w) seen[i] = ph + 1;
        return w;
    };
    if (tid == 0)
    {
        mbar_arrive_expect_tx(&bars[BQ], Sh::QBYTES);
        for (int j = 0; j < HD / 32; ++j)
            tma_load_2d(q_s + j * (QB * 128), &map_q, (int)(h * HD) + 32 * j, (int)(b * P + q0), &bars[BQ]);
        issued[BQ] = 1;
        issue_k(0);
        issue_v(0);
    }

    bool ok = wait(BQ, 0);
    if constexpr (SPLIT3)
        if (ok)
            lo_inplace(reinterpret_cast<float4*>(qlo_s), reinterpret_cast<const float4*>(q_s), Sh::QBYTES / 16, tid);

    float o[HD];
#pragma unroll
    for (int e = 0; e < HD; ++e) o[e] = 0.f;
    float m = -INFINITY, l = 0.f;

    for (uint32_t t = 0; t < ntiles; ++t)
    {
        const uint32_t k0 = t * KT;
        // ---- S = Q K^T ----
        if (ok) ok = wait(BKEY, t);
        if constexpr (SPLIT3)
            if (ok)
                lo_inplace(reinterpret_cast<float4*>(klo_s), reinterpret_cast<const float4*>(k_s), Sh::KBYTES / 16,
                           tid);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        ok = __syncthreads_and(ok) != 0;
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (warp0)
        {
#pragma unroll
            for (int j = 0; j < HD / 32; ++j)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                {
                    const uint64_t da = smem_desc(q_s + j * (QB * 128), kk * 32);
                    const uint64_t db = smem_desc(k_s + j * (KT * 128), kk * 32);
                    mma_tf32_elected(tmem, da, db, IDESC_S, j > 0 || kk > 0);
                    if constexpr (SPLIT3)
                    {
                        mma_tf32_elected(tmem, da, smem_desc(klo_s + j * (KT * 128), kk * 32), IDESC_S, true);
                        mma_tf32_elected(tmem, smem_desc(qlo_s + j * (QB * 128), kk * 32), db, IDESC_S, true);
                    }
                }
            mma_commit_elected(&bars[BS]);
            ++issued[BS];
        }
        ok = wait(BS, t);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        // the K tile is consumed: the next one's copy can start
        if (tid == 0 && ok && t + 1 < ntiles) issue_k(t + 1);

        // ---- row softmax (thread = query row) ----
        float sv[KT];
        if (ok)
        {
#pragma unroll
            for (int c = 0; c < KT; c += 32)
            {
                float v[32];
                tmem_ld32(tmem + lane_base + (uint32_t)c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) sv[c + i] = v[i];
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < KT; ++i) sv[i] = 0.f;
        }
        float mx = m;
#pragma unroll
        for (int i = 0; i < KT; ++i)
        {
            const uint32_t key = k0 + i;
            const bool live = key <= q && key < P;
            sv[i] = live ? sv[i] * a.scale : -INFINITY;  // a select: masked slots may hold anything
            mx = fmaxf(mx, sv[i]);
        }
        const float corr = m == -INFINITY ? 0.f : expf(m - mx);
        float psum = 0.f;
#pragma unroll
        for (int i = 0; i < KT; ++i)
        {
            sv[i] = sv[i] == -INFINITY ? 0.f : expf(sv[i] - mx);
            psum += sv[i];
        }
        l = l * corr + psum;
        m = mx;
        // P row into the K-major 128-byte-swizzled A tile: keys kb*32 + 4c ..
        // + 3 of row tid sit in 16-byte chunk c ^ (tid % 8) of the row
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
            for (int c = 0; c < 8; ++c)
            {
                const float4 pv = make_float4(sv[kb * 32 + 4 * c], sv[kb * 32 + 4 * c + 1], sv[kb * 32 + 4 * c + 2],
                                              sv[kb * 32 + 4 * c + 3]);
                const uint32_t off = kb * (QB * 128) + tid * 128 + ((c ^ (tid & 7)) * 16);
                *reinterpret_cast<float4*>(p_s + off) = pv;
                if constexpr (SPLIT3) *reinterpret_cast<float4*>(plo_s + off) = tf32_lo4(pv);
            }

        // ---- O_tile = P V ----
        if (ok) ok = wait(BVAL, t);
        if (ok)
        {
            // key rows past the last key any row of this CTA sees are zeroed
            // (the cache there may hold anything, and 0 * NaN is NaN); with
            // TF32x3 the same pass writes the lo part of the others.  Box
            // (kb, j) = keys kb*32.., head columns 32j.. is 4 KB of 32 rows.
            const uint32_t valid = nkeys - k0 < (uint32_t)KT ? nkeys - k0 : (uint32_t)KT;
            if (SPLIT3 || valid < (uint32_t)KT)
            {
                float4* v4 = reinterpret_cast<float4*>(v_s);
                float4* vlo4 = reinterpret_cast<float4*>(vlo_s);
                for (uint32_t i = tid; i < Sh::VBYTES / 16; i += 128)
                {
                    const uint32_t key = (i / 256) / (HD / 32) * 32 + (i % 256) / 8;
                    if (key >= valid)
                    {
                        v4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if constexpr (SPLIT3) vlo4[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                    else if constexpr (SPLIT3)
                        vlo4[i] = tf32_lo4(v4[i]);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        ok = __syncthreads_and(ok) != 0;
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (warp0)
        {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                {
                    const uint64_t da = smem_desc(p_s + kb * (QB * 128), kk * 32);
                    const uint64_t db = desc_mn(v_s + kb * (HD / 32) * 4096 + kk * 1024);
                    mma_tf32_elected(tmem_o, da, db, IDESC_O, kb > 0 || kk > 0);
                    if constexpr (SPLIT3)
                    {
                        mma_tf32_elected(tmem_o, da, desc_mn(vlo_s + kb * (HD / 32) * 4096 + kk * 1024), IDESC_O, true);
                        mma_tf32_elected(tmem_o, smem_desc(plo_s + kb * (QB * 128), kk * 32), db, IDESC_O, true);
                    }
                }
            mma_commit_elected(&bars[BO]);
            ++issued[BO];
        }
        ok = wait(BO, t);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (tid == 0 && ok && t + 1 < ntiles) issue_v(t + 1);  // the V tile and P are consumed
        if (ok)
        {
#pragma unroll
            for (int c = 0; c < HD; c += 32)
            {
                float v[32];
                tmem_ld32(tmem_o + lane_base + (uint32_t)c, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[c + i] = fmaf(o[c + i], corr, v[i]);
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    }
    ok = __syncthreads_and(ok) != 0;

    if (ok && q < P)
    {
        const float inv = 1.0f / l;  // l >= 1: the row's largest score contributes exp(0)
        float* dst = a.out + (uint64_t)(b * P + q) * a.ldo + h * HD;
#pragma unroll
        for (int e = 0; e < HD; e += 4)
            *reinterpret_cast<float4*>(dst + e) = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
    }
    if (!ok && tid == 0)
    {
        atomicAdd(&g_prefill_tc_timeouts, 1);
        // copies and products still in flight must land before the CTA frees
        // its shared memory and TMEM (bounded waits)
        for (int i = 0; i < 5; ++i)
            for (uint32_t ph = seen[i]; ph < issued[i]; ++ph) mbar_wait(&bars[i], ph & 1u);
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 0)
    {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Sh::TCOLS) : "memory");
    }
}

// ---- head dim 64: two query tiles per CTA, warp-specialised ---------------
//
// CTA = 12 warps on (256 query rows as two 128-row tiles A and B, head,
// sequence); the two tiles share every K / V tile, and their softmax and
// MMA phases interleave so that the tensor pipe works on one tile while the
// CUDA cores work on the other:
//   warps 0-3   softmax of tile A (thread = TMEM lane = query row)
//   warps 4-7   softmax of tile B
//   warp 8      converter: the TF32 lo parts of K and V (TF32x3) and the
//               zeroing of V rows past the last key any row sees
//   warps 9-10  tile A's / tile B's tcgen05.mma (one lane elected)
//   warp 11     one thread issues every TMA copy
// K and V operand tiles are double-buffered: the copy and the conversion of
// key tile t + 1 run while tile t's products do.
// TMEM per query tile (2 x 256 columns): S = Q K^T [64 keys | the hi.lo
// half], overwritten in place by P = exp(S - m) and P's lo part (the A
// operands of O += P V, read from TMEM); the O accumulator [64], which stays
// in TMEM over all key tiles; and Q's lo part [64] (the A operand of the
// lo.hi term of S).  A tf32 MMA of N = 64 costs 3/4 of one of N = 128 on
// this part (it runs the tensor pipe at 2/3 of its rate), so S's hi.hi and
// hi.lo terms are ONE MMA of N = 128 against [K hi | K lo] (the lo rows sit
// next to the hi rows of each K box); O's three terms stay 64 wide for the
// TMEM that Q lo needs.
// A row rescales O (tcgen05.ld / st) only when its running maximum rises by
// more than 2^8 over the one its P values were taken against, so P stays
// below 256 and fp32 keeps its precision; the result O / l does not depend
// on the reference maximum.
// The tensor pipe's instruction queue is short: while the thread that issues
// MMAs waits on an mbarrier (even one already complete, ~170 cycles), the
// pipe drains and idles.  So each query tile has its own issuing warp, and
// the pipe runs one tile's products while the other's
// warp waits (for its softmax, or for the completion of O_x(t-1): S_x(t)
// overwrites the columns P_x(t-1) is read from).
//
// PACKED: the same over packed prompts with grouped heads (packed.cuh) at head
// dims 32, 64 and 128: a CTA has ONE tile of (token, query head) rows of one
// key/value head, each with the number of keys that it sees, one buffer of K
// and of V, two softmax warps to a row, half of the keys each (their maxima
// meet in shared memory), and converters that also start the copies.  At head
// dims 32 and 64 two such CTAs share an SM, so that one's start, waits and end
// lie under the other's work: 64 ragged prompts of 8 heads of 64 took 67 us so,
// with the two tiles above and one CTA 84 us.  Head dim 128 has shared memory
// for one.
// Precision: the tensor cores cut their running sums, so a key tile's P V is a
// sum of its own, added to the row's in registers (kept in TMEM over all keys
// it is 1.6e-5 off after 3300 keys, so 5e-7, and 9 % faster); the small terms go
// into sums of their own (S) or first (P V); remainders are rounded to TF32.
// What bounds it: a step of 64 keys is a chain of S, softmax and P V of about
// 4500 cycles, the tensor cores' share 1536 at head dim 64; two CTAs overlap
// theirs only in part.  Measured on a B200, one causal prompt of 512 tokens: 4
// heads of 32 21 us, 8 of 64 26 us, 32 on 8 of 128 37 us (on the CUDA cores 43,
// 61 and 151 us; of 1 token 6.1 against 7.4, 7.3 against 10, 8.9 against 15: the
// tensor cores take every call whose alignment and scale they can).
// Every wait is bounded and also returns early once any role has recorded an
// expiry in the CTA's abort flag; the MMA thread then waits for its MMAs and
// the copy thread for its copies (bounded) before TMEM is freed.
namespace {

constexpr int PP_HD = 64, PP_KT = 64;  // head dim of the prompts of one length; keys of a tile
template <int HD, bool PACKED>
struct PpShape
{
    // two CTAs of an SM have 256 TMEM columns, half of the shared memory and 80 registers a thread each
    static constexpr int CTAS = PACKED && HD < 128 ? 2 : 1;  // on an SM
    static constexpr int NX = PACKED ? 1 : 2, NB = PACKED ? 1 : 2;
    static constexpr int SPLIT = PACKED ? 2 : 1;             // softmax warps that share a row's keys
    // warps: 4 NX SPLIT of softmax, then the converters (PACKED: their first lane copies too), NX that
    // issue the MMAs, and without PACKED one that copies
    static constexpr int SM = 4 * NX * SPLIT, CW = !PACKED || HD == 32 ? 1 : HD == 64 ? 2 : 4, MMA = SM + CW, TMA = MMA + NX;
    static constexpr int THREADS = 32 * (TMA + !PACKED);
    static constexpr uint32_t CONV = 32 * CW;               // converter threads
    static constexpr uint32_t QTILE = 128 * HD * 4;         // one 128-row Q tile
    static constexpr uint32_t KVT = PP_KT * HD * 4;         // one K or V tile
    // operand tiles: K box j (head columns 32j..) = [64 hi rows | 64 lo rows] of
    // 128 bytes (16 KB); V key block kb = 4 KB boxes of 32 keys [hi columns 0-31,
    // hi 32-63 .., lo 0-31 ..]
    static constexpr uint32_t KBOX = 2 * PP_KT * 128, VLO = HD / 32 * 4096, VBLK = 2 * VLO, KVOP = 2 * KVT;
    // Q hi tiles, then NB K and NB V operand tiles (hi and lo each)
    static constexpr uint32_t SMEM = NX * QTILE + 2 * NB * KVOP + 1024 + 256;
    // TMEM columns of tile x: S / P [0, 64), S's hi.lo half / P lo [64, 128), O, Q lo
    static constexpr uint32_t TX = 256, PLO = 64, O = 128, QLO = 128 + HD, COLS = CTAS == 2 ? 256 : 512;
};
// per operand buffer b: F copy landed, R converted, E[x] consumed by tile
// x's MMAs (index 2x + b); per query tile x: S, P, O and the final drain
enum PpBar { PB_QF, PB_QR, PB_KF, PB_KR = PB_KF + 2, PB_KE = PB_KR + 2, PB_VF = PB_KE + 4, PB_VR = PB_VF + 2,
             PB_VE = PB_VR + 2, PB_S0 = PB_VE + 4, PB_P0 = PB_S0 + 2, PB_O0 = PB_P0 + 2, PB_FIN = PB_O0 + 2,
             PB_N = PB_FIN + 2 };

}  // namespace

template <int HD, bool SPLIT3, bool PACKED>
__global__ void __launch_bounds__(PpShape<HD, PACKED>::THREADS, PpShape<HD, PACKED>::CTAS)
    prefill_attention_pp_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                const __grid_constant__ CUtensorMap map_v, PfArgs a, PackedArgs pk)
{
    using namespace tc;
    using Pp = PpShape<HD, PACKED>;
    constexpr int NX = Pp::NX, NB = Pp::NB;
    constexpr uint32_t IDESC_S = idesc_tf32(128, PP_KT);
    constexpr uint32_t IDESC_S2 = idesc_tf32(128, 2 * PP_KT);          // [K hi | K lo]
    constexpr uint32_t IDESC_O = idesc_tf32(128, HD) | (1u << 16);     // B (V) read MN-major
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem =
        reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* q_s = smem;                    // Q hi of tile x at x * QTILE
    unsigned char* k_op = smem + NX * Pp::QTILE;  // K operand buffer b at b * KVOP (Pp::KBOX layout)
    unsigned char* v_op = k_op + NB * Pp::KVOP;   // V operand buffer b at b * KVOP (Pp::VBLK layout)
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_op + NB * Pp::KVOP);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + PB_N);
    volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // heaviest query blocks (most key tiles) first
    const uint32_t qblk = gridDim.x - 1 - blockIdx.x;
    const uint32_t q0 = qblk * 256, h = PACKED ? blockIdx.x % (pk.kv_heads * pk.nchunk) : blockIdx.y, b = blockIdx.z;
    const uint32_t P = a.P;
    bool has_b = q0 + 128 < P;
    // the keys that tile A's rows see, and any row of the CTA
    uint32_t nkeys0 = min(q0 + 128u, P), nkeys = min(q0 + 256u, P);
    int kv_row0 = (int)((b * a.H + h) * a.C), kv_col0 = 0;
    PackedTile pt{};
    uint32_t kvh = 0, hc = 0, tokens = 0;  // PACKED: heads, tokens of the tile
    if constexpr (PACKED)
    {
        __shared__ PackedTile found;
        if (warp == 0)
        {
            const PackedTile t = packed_tile(pk, packed_totals(pk), blockIdx.x / (pk.kv_heads * pk.nchunk));
            if (lane == 0) found = t;
        }
        __syncthreads();
        pt = found;
        if (!pt.live) return;
        kvh = h / pk.nchunk;
        hc = (h % pk.nchunk) * pk.gs;
        tokens = min(pk.tpt, pt.lq - pt.t0);
        has_b = false;
        nkeys0 = nkeys = keys_seen(pt, pt.t0 + tokens - 1);
        kv_row0 = (int)pt.k0;
        kv_col0 = (int)(kvh * HD);
    }
    // key tiles of tile A / B
    const uint32_t nt0 = (nkeys0 + PP_KT - 1) / PP_KT;
    const uint32_t nt1 = has_b ? (nkeys + PP_KT - 1) / PP_KT : 0u;
    const uint32_t ntiles = has_b ? nt1 : nt0;

    if (tid == 0)
    {
        for (int i = 0; i < PB_N; ++i)
        {
            uint32_t count = 1;
            if (i == PB_QR) count = 32 * Pp::SM;  // every softmax thread writes its Q lo row
            if (i == PB_KR || i == PB_KR + 1 || i == PB_VR || i == PB_VR + 1) count = Pp::CONV;
            if (i == PB_P0 || i == PB_P0 + 1) count = 128 * Pp::SPLIT;
            mbar_init(&bars[i], count);
        }
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(Pp::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp < Pp::SM)
    {
        // ---------------- softmax of tile x: keys c0 .. c0 + KS - 1 of its key tiles ----------------
        constexpr int SPLIT = Pp::SPLIT, KS = PP_KT / SPLIT, OS = HD / SPLIT;
        const int x = SPLIT == 1 ? warp >> 2 : 0, part = SPLIT == 1 ? 0 : warp >> 2;
        const int c0 = part * KS, o0 = part * OS;  // its keys; the output columns that it scales and writes
        __shared__ float row_max[SPLIT][2][128], row_sum[SPLIT][128];
        // the other warp of the row: both come here equally often, whatever became of their waits
        auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp & 3)) : "memory"); };
        const uint32_t nt = x ? nt1 : nt0;
        const int r = 32 * (warp & 3) + lane;                 // row within the tile
        const uint32_t row = q0 + 128u * x + (uint32_t)r;     // this thread's query row
        uint32_t seen = 0, least = 0, q_row = b * P + row, q_head = h;  // PACKED: keys it sees, the warp's least
        bool live = row < P;
        if constexpr (PACKED)
        {
            const uint32_t tok = (uint32_t)r / pk.gs, head = (uint32_t)r % pk.gs;
            live = tok < tokens && head < min(pk.gs, pk.group - hc);
            const uint32_t token = pt.t0 + tok;
            seen = live ? keys_seen(pt, token) : 0xffffffffu;  // rows that are no query's are left unmasked
            least = __reduce_min_sync(FULL_MASK, seen);
            q_row = pt.q0 + token;
            q_head = kvh * pk.group + hc + head;
        }
        const uint32_t tx = tmem + Pp::TX * x + ((uint32_t)(32 * (warp & 3)) << 16);
        const float sl2 = a.scale * 1.4426950408889634f;  // scores in log2 units
        float m = -INFINITY, l = 0.f;
        // PACKED: the key tiles' P V, added here: the tensor cores cut their running sums, and the
        // error would grow with the keys
        float acc[PACKED ? OS : 1];
#pragma unroll
        for (int i = 0; i < (PACKED ? OS : 1); ++i) acc[i] = 0.f;
        auto add_tile = [&] {
#pragma unroll
            for (int c = 0; c < OS; c += 16)
            {
                float v[16];
                tmem_ld16(tx + Pp::O + o0 + c, v);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[PACKED ? c + i : 0] += v[i];
            }
        };
        bool ok = __all_sync(FULL_MASK, mbar_wait_or(&bars[PB_QF], 0, abort));
        if (ok && SPLIT3)
        {
            // Q lo of this row into TMEM: row r of box j holds head columns
            // 32j + 4c.. in 16-byte chunk c ^ (r % 8)
            const unsigned char* qrow = q_s + x * Pp::QTILE + r * 128;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j)
            {
                if (SPLIT == 2 && (j & 1) != part) continue;
                uint32_t u[32];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                {
                    const float4 v = *reinterpret_cast<const float4*>(qrow + j * (128 * 128) + ((c ^ (r & 7)) * 16));
                    const float4 lo = tf32_lo4_as<PACKED>(v);
                    u[4 * c] = __float_as_uint(lo.x);
                    u[4 * c + 1] = __float_as_uint(lo.y);
                    u[4 * c + 2] = __float_as_uint(lo.z);
                    u[4 * c + 3] = __float_as_uint(lo.w);
                }
                tmem_st32(tx + Pp::QLO + 32 * j, u);
            }
            tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(&bars[PB_QR]);
        for (uint32_t t = 0; SPLIT == 2 ? t < nt : ok && t < nt; ++t)
        {
            ok = ok && __all_sync(FULL_MASK, mbar_wait_or(&bars[PB_S0 + x], t, abort));
            if (SPLIT == 1 && !ok) break;
            float s[KS], mt = -INFINITY;
            if (ok)
            {
                tc_fence_after();
                // O_x(t-1) has completed: S_x(t) was issued after it
                if (PACKED && t > 0) add_tile();
                if constexpr (PACKED)
                {
                    static_assert(KS == 32, "");
                    tmem_ld32(tx + c0, s);
                    if constexpr (SPLIT3)
#pragma unroll
                        for (int c = 0; c < KS; c += 16)
                        {
                            float w[16];
                            tmem_ld16(tx + Pp::PLO + c0 + c, w);
#pragma unroll
                            for (int i = 0; i < 16; ++i) s[c + i] += w[i];
                        }
                }
                else
                {
#pragma unroll
                    for (int c = 0; c < KS; c += 32)
                    {
                        uint32_t u[32];
                        tmem_ld32_async(tx + c0 + c, u);
                        if constexpr (SPLIT3)
                        {
                            uint32_t w[32];
                            tmem_ld32_async(tx + Pp::PLO + c0 + c, w);
                            tmem_wait_ld(u);
                            tmem_wait_ld(w);
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[c + i] = __uint_as_float(u[i]) + __uint_as_float(w[i]);
                        }
                        else
                        {
                            tmem_wait_ld(u);
#pragma unroll
                            for (int i = 0; i < 32; ++i) s[c + i] = __uint_as_float(u[i]);
                        }
                    }
                }
                const uint32_t k0 = t * PP_KT + c0;
                // the mask only bites in tiles that reach past the warp's first
                // row or past the prompt (a warp-uniform test)
                const uint32_t row0 = row - lane;
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (PACKED ? k0 + KS <= least : k0 + KS - 1 <= row0 && k0 + KS <= P)
                {
#pragma unroll
                    for (int i = 0; i < KS; ++i)
                    {
                        s[i] *= sl2;
                        mx4[i & 3] = fmaxf(mx4[i & 3], s[i]);
                    }
                }
                else
                {
#pragma unroll
                    for (int i = 0; i < KS; ++i)
                    {
                        const uint32_t key = k0 + i;
                        const bool in = PACKED ? key < seen : key <= row && key < P;
                        s[i] = in ? s[i] * sl2 : -INFINITY;  // a select: masked slots may hold NaN
                        mx4[i & 3] = fmaxf(mx4[i & 3], s[i]);
                    }
                }
                mt = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            }
            if constexpr (SPLIT == 2)
            {
                row_max[part][t & 1u][r] = mt;
                meet();
                mt = fmaxf(mt, row_max[part ^ 1][t & 1u][r]);
                if (!ok) continue;
            }
            const bool need = mt > m + 8.0f;
            if (__any_sync(FULL_MASK, need))
            {
                const float mn = need ? mt : m;
                const float corr = need ? ex2_approx(m - mn) : 1.f;  // 0 on the first tile (m = -inf)
                l *= corr;
                m = mn;
                if constexpr (PACKED)
                {
#pragma unroll
                    for (int i = 0; i < OS; ++i) acc[i] *= corr;
                }
                else if (t > 0)
                {
                    // O_x(t-1) has completed: S_x(t) was issued after it
#pragma unroll
                    for (int c = 0; c < HD; c += 32)
                    {
                        float v[32];
                        uint32_t u[32];
                        tmem_ld32(tx + Pp::O + c, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(v[i] * corr);
                        tmem_st32(tx + Pp::O + c, u);
                    }
                }
            }
            float ls[4] = {0.f, 0.f, 0.f, 0.f};
            const float base = PACKED && m == -INFINITY ? 0.f : m;  // a packed row may see no key
#pragma unroll
            for (int c = 0; c < KS; c += 32)
            {
                uint32_t u[32];
#pragma unroll
                for (int i = 0; i < 32; ++i)
                {
                    const float p = ex2_approx(s[c + i] - base);  // 0 for masked keys
                    ls[i & 3] += p;
                    s[c + i] = p;
                    u[i] = __float_as_uint(p);
                }
                tmem_st32(tx + c0 + c, u);  // P over S's columns (the MMA reads its TF32 part)
                if constexpr (SPLIT3 && PACKED)
#pragma unroll
                    for (int h = 0; h < 32; h += 16)
                    {
                        uint32_t w[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(tf32_lo<PACKED>(s[c + h + i]));
                        tmem_st16(tx + Pp::PLO + c0 + c + h, w);
                    }
                else if constexpr (SPLIT3)
                {
#pragma unroll
                    for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(tf32_lo<PACKED>(s[c + i]));
                    tmem_st32(tx + Pp::PLO + c0 + c, u);
                }
            }
            l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bars[PB_P0 + x]);
        }
        if constexpr (SPLIT == 2)
        {
            row_sum[part][r] = l;
            meet();
            l = row_sum[0][r] + row_sum[1][r];
        }
        if (ok && nt > 0)
        {
            ok = __all_sync(FULL_MASK, mbar_wait_or(&bars[PB_O0 + x], nt - 1, abort));
            if (ok)
            {
                tc_fence_after();
                const float inv = 1.0f / l;
                float* dst = a.out + (uint64_t)q_row * a.ldo + (uint64_t)q_head * HD + o0;
                if constexpr (PACKED)
                {
                    add_tile();
#pragma unroll
                    for (int i = 0; i < OS; ++i) acc[i] = seen == 0 ? 0.f : acc[i] * inv;
                    if (live)
#pragma unroll
                        for (int i = 0; i < OS; i += 4)
                            *reinterpret_cast<float4*>(dst + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
                }
                else
                {
#pragma unroll
                    for (int c = 0; c < HD; c += 32)
                    {
                        float v[32];
                        tmem_ld32(tx + Pp::O + c, v);
                        if (live)
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<float4*>(dst + c + i) =
                                    make_float4(v[i] * inv, v[i + 1] * inv, v[i + 2] * inv, v[i + 3] * inv);
                    }
                }
            }
        }
        if (PACKED && ok && nt == 0 && live)
        {
            float* dst = a.out + (uint64_t)q_row * a.ldo + (uint64_t)q_head * HD;
            for (int i = o0; i < o0 + OS; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    else if (warp < Pp::MMA)
    {
        // ---------------- converter ----------------
        constexpr int NK = 512 / Pp::CONV, NV = HD / 32 * 256 / Pp::CONV;  // float4 of a box, of a block, each
        const int ct = tid - 32 * Pp::SM;
        // K: lo rows from the hi rows the copy wrote (box j = 512 float4 hi, then 512 lo)
        auto convert_k = [&](uint32_t bf) {
            if constexpr (SPLIT3)
            {
                // loads in flight before the stores
#pragma unroll
                for (int c = 0; c < HD / 32; ++c)
                {
                    float4* box = reinterpret_cast<float4*>(k_op + bf * Pp::KVOP + c * Pp::KBOX);
                    float4 v[NK];
#pragma unroll
                    for (int n = 0; n < NK; ++n) v[n] = box[ct + Pp::CONV * n];
#pragma unroll
                    for (int n = 0; n < NK; ++n) box[512 + ct + Pp::CONV * n] = tf32_lo4_as<PACKED>(v[n]);
                }
            }
            fence_async_smem();
            mbar_arrive(&bars[PB_KR + bf]);
        };
        // V(t): key block kb = hi boxes (256 float4 each) then lo boxes; rows at or
        // past `nkeys` are zeroed (the cache there may hold anything, and 0 * NaN is NaN)
        auto convert_v = [&](uint32_t bf, uint32_t t) {
            const uint32_t k0 = t * PP_KT;
            const uint32_t valid = nkeys - k0 < (uint32_t)PP_KT ? nkeys - k0 : (uint32_t)PP_KT;
#pragma unroll
            for (int c = 0; c < PP_KT / 32; ++c)
            {
                float4* blk = reinterpret_cast<float4*>(v_op + bf * Pp::KVOP + c * Pp::VBLK);
                if (valid == (uint32_t)PP_KT)
                {
                    if constexpr (SPLIT3)
                    {
                        float4 v[NV];
#pragma unroll
                        for (int n = 0; n < NV; ++n) v[n] = blk[ct + Pp::CONV * n];
#pragma unroll
                        for (int n = 0; n < NV; ++n) blk[Pp::VLO / 16 + ct + Pp::CONV * n] = tf32_lo4_as<PACKED>(v[n]);
                    }
                }
                else
                {
                    for (int n = 0; n < NV; ++n)
                    {
                        const uint32_t i = ct + Pp::CONV * n, key = c * 32 + (i % 256) / 8;
                        if (key >= valid)
                        {
                            blk[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if constexpr (SPLIT3) blk[Pp::VLO / 16 + i] = make_float4(0.f, 0.f, 0.f, 0.f);
                        }
                        else if constexpr (SPLIT3)
                            blk[Pp::VLO / 16 + i] = tf32_lo4_as<PACKED>(blk[i]);
                    }
                }
            }
            fence_async_smem();
            mbar_arrive(&bars[PB_VR + bf]);
        };
        if constexpr (PACKED)
        {
            // one buffer of each: K(t + 1) is copied and converted while the softmax of
            // tile t runs, V(t + 1) while that of tile t + 1 does (both copies before both
            // conversions was slower: the first conversion then waits for S)
            static_assert(NB == 1, "");
            uint32_t nk = 0, nv = 0;  // copies of each that the first thread has started
            auto copy_k = [&](uint32_t t) {
                mbar_arrive_expect_tx(&bars[PB_KF], Pp::KVT);
                for (int j = 0; j < HD / 32; ++j)
                    tma_load_2d(k_op + j * Pp::KBOX, &map_k, kv_col0 + 32 * j, kv_row0 + (int)(t * PP_KT), &bars[PB_KF]);
                ++nk;
            };
            auto copy_v = [&](uint32_t t) {
                mbar_arrive_expect_tx(&bars[PB_VF], Pp::KVT);
                for (int kb = 0; kb < PP_KT / 32; ++kb)
                    for (int j = 0; j < HD / 32; ++j)
                        tma_load_2d(v_op + kb * Pp::VBLK + j * 4096, &map_v, kv_col0 + 32 * j,
                                    kv_row0 + (int)(t * PP_KT) + 32 * kb, &bars[PB_VF]);
                ++nv;
            };
            if (ct == 0)
            {
                mbar_arrive_expect_tx(&bars[PB_QF], HD / 32 * pk.gs * pk.tpt * 128);
                for (int j = 0; j < HD / 32; ++j)
                    tma_load_3d(q_s + j * (128 * 128), &map_q, 32 * j, (int)(kvh * pk.group + hc),
                                (int)(pt.q0 + pt.t0), &bars[PB_QF]);
                if (nt0 > 0) copy_k(0), copy_v(0);
            }
            for (uint32_t t = 0; t < nt0; ++t)
            {
                if (ct == 0 && t > 0)
                {
                    if (!mbar_wait_or(&bars[PB_KE], t - 1, abort)) break;
                    copy_k(t);
                }
                if (!mbar_wait_or(&bars[PB_KF], t, abort)) break;
                convert_k(0);
                if (ct == 0 && t > 0)
                {
                    if (!mbar_wait_or(&bars[PB_VE], t - 1, abort)) break;
                    copy_v(t);
                }
                if (!mbar_wait_or(&bars[PB_VF], t, abort)) break;
                convert_v(0, t);
            }
            if (ct == 0)
            {
                // the copies that this thread started land before the CTA exits (bounded; immediate
                // on the normal path)
                mbar_wait(&bars[PB_QF], 0);
                if (nk) mbar_wait(&bars[PB_KF], (nk - 1) & 1u);
                if (nv) mbar_wait(&bars[PB_VF], (nv - 1) & 1u);
            }
        }
        else
            for (uint32_t t = 0; t < ntiles; ++t)
            {
                const uint32_t bf = t % NB, ph = t / NB;
                if (!mbar_wait_or(&bars[PB_KF + bf], ph, abort)) break;
                convert_k(bf);
                if (!mbar_wait_or(&bars[PB_VF + bf], ph, abort)) break;
                convert_v(bf, t);
            }
    }
    else if (warp < Pp::TMA)
    {
        // ---------------- MMA issue for tile x ----------------
        const int x = __shfl_sync(FULL_MASK, warp, 0) - Pp::MMA;  // the same in the warp for the compiler too
        const uint32_t nt = x ? nt1 : nt0;
        if (nt > 0)
        {
            auto wait = [&](int i, uint32_t ph) { return __all_sync(FULL_MASK, mbar_wait_or(&bars[i], ph, abort)) != 0; };
            // descriptors: one base each, advanced by (byte offset >> 4) in
            // the start-address field (shared addresses stay below 2^18)
            const uint64_t dq = smem_desc(q_s + x * Pp::QTILE, 0);
            const uint64_t dk = smem_desc(k_op, 0), dv = desc_mn(v_op);
            const uint32_t ts = tmem + Pp::TX * x, to = ts + Pp::O;
            bool ok = wait(PB_QR, 0);
            for (uint32_t t = 0; ok && t < nt; ++t)
            {
                const uint32_t bf = t % NB, ph = t / NB;
                // S_x(t) = Q_x K(t)^T, after O_x(t-1) has read P_x(t-1)
                if (!(ok = wait(PB_KR + bf, ph))) break;
                if (t > 0 && !(ok = wait(PB_O0 + x, t - 1))) break;
                tc_fence_after();
                const uint64_t kbase = dk + ((bf * Pp::KVOP) >> 4);
#pragma unroll
                for (int j = 0; j < HD / 32; ++j)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                    {
                        const uint64_t da = dq + ((j * (128 * 128) + kk * 32) >> 4);
                        const uint64_t db = kbase + ((j * Pp::KBOX + kk * 32) >> 4);
                        if constexpr (SPLIT3)
                        {
                            // [hi.hi | hi.lo] in one MMA, then lo.hi (Q lo from TMEM) into the first half
                            mma_tf32_elected(ts, da, db, IDESC_S2, j > 0 || kk > 0);
                            // (PACKED: into the second, which keeps cuts of its sum off the large one)
                            mma_tf32_tmem_a_elected(ts + (PACKED ? Pp::PLO : 0u), ts + Pp::QLO + 32 * j + 8 * kk, db,
                                                    IDESC_S, true);
                        }
                        else
                            mma_tf32_elected(ts, da, db, IDESC_S, j > 0 || kk > 0);
                    }
                mma_commit_elected(&bars[PB_S0 + x]);
                mma_commit_elected(&bars[PB_KE + 2 * x + bf]);
                // O_x += P_x(t) V(t)
                if (!(ok = wait(PB_VR + bf, ph))) break;
                if (!(ok = wait(PB_P0 + x, t))) break;
                tc_fence_after();
                const uint64_t vbase = dv + ((bf * Pp::KVOP) >> 4);
                // PACKED: the small terms of all keys first, so that fewer sums of full size are cut
#pragma unroll
                for (int part = 0; part < (PACKED && SPLIT3 ? 2 : 1); ++part)
#pragma unroll
                    for (int kb = 0; kb < PP_KT / 32; ++kb)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                        {
                            const uint64_t db = vbase + ((kb * Pp::VBLK + kk * 1024) >> 4);
                            const uint32_t col = kb * 32 + kk * 8;
                            const bool more = (!PACKED && t > 0) || kb > 0 || kk > 0;
                            if (!PACKED || !SPLIT3 || part == 1)
                                mma_tf32_tmem_a_elected(to, ts + col, db, IDESC_O, more || part == 1);
                            if (SPLIT3 && part == 0)
                            {
                                mma_tf32_tmem_a_elected(to, ts + col, db + (Pp::VLO >> 4), IDESC_O,
                                                        more || !PACKED);                             // P hi . V lo
                                mma_tf32_tmem_a_elected(to, ts + Pp::PLO + col, db, IDESC_O, true);  // P lo . V hi
                            }
                        }
                mma_commit_elected(&bars[PB_O0 + x]);
                mma_commit_elected(&bars[PB_VE + 2 * x + bf]);
            }
            // every MMA this warp issued completes before TMEM is freed
            mma_commit_elected(&bars[PB_FIN + x]);
            __all_sync(FULL_MASK, mbar_wait(&bars[PB_FIN + x], 0));
        }
    }
    else if constexpr (!PACKED)
    {
        // ---------------- TMA copies ----------------
        if (lane == 0)
        {
            const int nq = has_b ? 2 : 1;
            mbar_arrive_expect_tx(&bars[PB_QF], nq * Pp::QTILE);
            for (int x = 0; x < nq; ++x)
                for (int j = 0; j < HD / 32; ++j)
                    tma_load_2d(q_s + x * Pp::QTILE + j * (128 * 128), &map_q, (int)(h * HD) + 32 * j,
                                (int)(b * P + q0 + 128 * x), &bars[PB_QF]);
            uint32_t issued = 0;
            for (uint32_t t = 0; t < ntiles; ++t)
            {
                const uint32_t bf = t % NB, ph = t / NB;
                // K(t) into buffer t % NB once S_A(t-NB) and S_B(t-NB) have read it
                const bool again = t >= NB;
                if (again && t - NB < nt0 && !mbar_wait_or(&bars[PB_KE + bf], ph - 1, abort)) break;
                if (again && t - NB < nt1 && !mbar_wait_or(&bars[PB_KE + 2 + bf], ph - 1, abort)) break;
                mbar_arrive_expect_tx(&bars[PB_KF + bf], Pp::KVT);
                for (int j = 0; j < HD / 32; ++j)
                    tma_load_2d(k_op + bf * Pp::KVOP + j * Pp::KBOX, &map_k, 32 * j, kv_row0 + (int)(t * PP_KT),
                                &bars[PB_KF + bf]);
                // V(t) once O_A(t-NB) and O_B(t-NB) have
                if ((again && t - NB < nt0 && !mbar_wait_or(&bars[PB_VE + bf], ph - 1, abort)) ||
                    (again && t - NB < nt1 && !mbar_wait_or(&bars[PB_VE + 2 + bf], ph - 1, abort)))
                {
                    issued = 2 * t + 1;
                    break;
                }
                mbar_arrive_expect_tx(&bars[PB_VF + bf], Pp::KVT);
                for (int kb = 0; kb < PP_KT / 32; ++kb)
                    for (int j = 0; j < HD / 32; ++j)
                        tma_load_2d(v_op + bf * Pp::KVOP + kb * Pp::VBLK + j * 4096, &map_v, 32 * j,
                                    kv_row0 + (int)(t * PP_KT) + 32 * kb, &bars[PB_VF + bf]);
                issued = 2 * t + 2;
            }
            // the copies this thread started land before the CTA exits
            // (bounded; immediate on the normal path).  Copy n < issued is
            // K(n / 2) for even n, V(n / 2) for odd n.
            mbar_wait(&bars[PB_QF], 0);
            for (uint32_t n = issued >= 2 * NB ? issued - 2 * NB : 0; n < issued; ++n)
            {
                const uint32_t t = n >> 1;
                mbar_wait(&bars[(n & 1u ? PB_VF : PB_KF) + t % NB], (t / NB) & 1u);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (tid == 0 && *abort) atomicAdd(&g_prefill_tc_timeouts, 1);
    if (warp == 0)
    {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Pp::COLS) : "memory");
    }
}

namespace {

template <int HD, bool SPLIT3>
int launch_tc_hd(const float* q, uint32_t ldq, const float* kc, const float* vc, uint32_t C, float* out, uint32_t ldo,
                 uint32_t B, uint32_t H, uint32_t P, float scale, cudaStream_t st)
{
    using Sh = PfShape<HD>;
    auto kern = prefill_attention_tc_kernel<HD, SPLIT3>;
    static uint64_t attr_devices = 0;
    FML_RC(smem_limit_once(reinterpret_cast<const void*>(kern), (int)Sh::SMEM, attr_devices));
    CUtensorMap mq, mk, mv;
    const uint64_t rows = (uint64_t)B * H * C;
    FML_REQUIRE(rows < (1ull << 31) && (uint64_t)B * P < (1ull << 31), "prefill attention: %llu cache rows",
                (unsigned long long)rows);
    FML_RC(tc::make_map(&mq, q, (int)(B * P), (int)(H * HD), (int)ldq, QB));
    FML_RC(tc::make_map(&mk, kc, (int)rows, HD, HD, Sh::KT));
    FML_RC(tc::make_map(&mv, vc, (int)rows, HD, HD, 32, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B));
    PfArgs a{out, ldo, B, H, P, C, scale};
    dim3 grid((P + QB - 1) / QB, H, B);
    kern<<<grid, 128, Sh::SMEM, st>>>(mq, mk, mv, a);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

template <bool SPLIT3>
int launch_pp(const float* q, uint32_t ldq, const float* kc, const float* vc, uint32_t C, float* out, uint32_t ldo,
              uint32_t B, uint32_t H, uint32_t P, float scale, cudaStream_t st)
{
    constexpr uint32_t SMEM = PpShape<PP_HD, false>::SMEM;
    auto kern = prefill_attention_pp_kernel<PP_HD, SPLIT3, false>;
    static uint64_t attr_devices = 0;
    FML_RC(smem_limit_once(reinterpret_cast<const void*>(kern), (int)SMEM, attr_devices));
    CUtensorMap mq, mk, mv;
    const uint64_t rows = (uint64_t)B * H * C;
    FML_REQUIRE(rows < (1ull << 31) && (uint64_t)B * P < (1ull << 31), "prefill attention: %llu cache rows",
                (unsigned long long)rows);
    FML_RC(tc::make_map(&mq, q, (int)(B * P), (int)(H * PP_HD), (int)ldq, 128));
    FML_RC(tc::make_map(&mk, kc, (int)rows, PP_HD, PP_HD, PP_KT));
    FML_RC(tc::make_map(&mv, vc, (int)rows, PP_HD, PP_HD, 32, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B));
    PfArgs a{out, ldo, B, H, P, C, scale};
    dim3 grid((P + 255) / 256, H, B);
    kern<<<grid, PpShape<PP_HD, false>::THREADS, SMEM, st>>>(mq, mk, mv, a, PackedArgs{});
    FML_LAUNCH_CHECK();
    return FML_OK;
}

// Packed prompts.
template <int HD, bool SPLIT3>
int launch_packed(float* out, const float* q, const float* k, const float* v, PackedArgs p, cudaStream_t st)
{
    using Pp = PpShape<HD, true>;
    auto kern = prefill_attention_pp_kernel<HD, SPLIT3, true>;
    static uint64_t attr_devices = 0;
    FML_RC(smem_limit_once(reinterpret_cast<const void*>(kern), (int)Pp::SMEM, attr_devices));
    const uint64_t blocks = packed_items(&p, 128, 1);
    FML_REQUIRE(blocks < (1ull << 31), "fml_attention_packed: %u rows, %u heads", p.q_rows, p.heads);
    CUtensorMap mq, mk, mv;
    FML_RC(tc::make_map_heads(&mq, q, HD, p.heads, p.q_rows, p.ldq, p.gs, p.tpt));
    FML_RC(tc::make_map(&mk, k, (int)p.k_rows, (int)(p.kv_heads * HD), (int)p.ldk, PP_KT));
    FML_RC(tc::make_map(&mv, v, (int)p.k_rows, (int)(p.kv_heads * HD), (int)p.ldv, 32, CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B));
    const PfArgs a{out, p.ldo, 0, 0, 0, 0, p.scale};
    kern<<<(unsigned)blocks, Pp::THREADS, Pp::SMEM, st>>>(mq, mk, mv, a, p);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

}  // namespace

// The packed prompt attention on fp32 inputs; FML_ERR_UNSUPPORTED (no error
// recorded) for bases or strides that TMA does not take, or no key row at all.
int launch_packed_attention_tf32(float* out, const float* q, const float* k, const float* v, uint32_t hd,
                                 const PackedArgs& p, bool split3, cudaStream_t st)
{
    if (p.k_rows == 0 || !aligned16(out) || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
        (p.ldo | p.ldq | p.ldk | p.ldv) % 4 || p.ldk > (1u << 30) || p.ldv > (1u << 30))
        return FML_ERR_UNSUPPORTED;
    if (split3)
    {
        if (hd == 32) return launch_packed<32, true>(out, q, k, v, p, st);
        if (hd == 64) return launch_packed<64, true>(out, q, k, v, p, st);
        return launch_packed<128, true>(out, q, k, v, p, st);
    }
    if (hd == 32) return launch_packed<32, false>(out, q, k, v, p, st);
    if (hd == 64) return launch_packed<64, false>(out, q, k, v, p, st);
    return launch_packed<128, false>(out, q, k, v, p, st);
}

// The tensor-core prefill attention.  q / out [B*P x ld] (head h at columns
// h*hd); keys and values of sequence b, head h at kc/vc + b*seq_stride +
// h*C*hd, rows 0..P-1 filled.  split3: TF32x3 (fp32-level), else one TF32
// product.  FML_ERR_UNSUPPORTED (no error recorded) for the layouts it does
// not take -- head dims other than 32 / 64 / 128, a cache whose sequences are
// not packed back to back, unaligned pointers or strides -- and the caller
// then uses the CUDA-core kernel.
int launch_prefill_attention_tc(const float* q, uint32_t ldq, const float* kc, const float* vc, uint64_t seq_stride,
                                uint32_t C, float* out, uint32_t ldo, uint32_t B, uint32_t H, uint32_t P, uint32_t hd,
                                float scale, bool split3, cudaStream_t st)
{
    if (!(hd == 32 || hd == 64 || hd == 128) || seq_stride != (uint64_t)H * C * hd || ldq % 4 || ldo % 4 ||
        !aligned16(q) || !aligned16(kc) || !aligned16(vc) || !aligned16(out) || B > 65535u || H > 65535u || P == 0)
        return FML_ERR_UNSUPPORTED;
    // FML_PREFILL_ATTN_SIMPLE=1: the one-tile kernel at head dim 64 as well
    // (tests run both)
    const char* simple = getenv("FML_PREFILL_ATTN_SIMPLE");
    if (hd == 64 && !(simple && simple[0] == '1'))
        return split3 ? launch_pp<true>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st)
                      : launch_pp<false>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
    if (split3)
    {
        if (hd == 32) return launch_tc_hd<32, true>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
        if (hd == 64) return launch_tc_hd<64, true>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
        return launch_tc_hd<128, true>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
    }
    if (hd == 32) return launch_tc_hd<32, false>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
    if (hd == 64) return launch_tc_hd<64, false>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
    return launch_tc_hd<128, false>(q, ldq, kc, vc, C, out, ldo, B, H, P, scale, st);
}

int launch_prefill_attention(const float* q, uint32_t ldq, const float* kc, const float* vc, uint64_t seq_stride,
                             uint32_t C, float* out, uint32_t ldo, uint32_t B, uint32_t H, uint32_t P, uint32_t hd,
                             float scale, cudaStream_t st);

int prefill_tc_error_count(int* out)
{
    FML_CUDA_TRY(cudaMemcpyFromSymbol(out, g_prefill_tc_timeouts, sizeof(int)));
    return FML_OK;
}

}  // namespace fml

using namespace fml;

extern "C" FML_API int fml_attention_prefill(float* out, const float* q, const float* kcache, const float* vcache,
                                             uint32_t batch, uint32_t heads, uint32_t head_dim, uint32_t context,
                                             uint32_t prompt_len, float scale, int mode, fml_stream_t stream)
{
    if (batch == 0 || prompt_len == 0) return FML_OK;
    FML_REQUIRE(out && q && kcache && vcache, "fml_attention_prefill: null pointer");
    FML_REQUIRE(heads >= 1 && prompt_len <= context, "fml_attention_prefill: %u heads, prompt %u, context %u", heads,
                prompt_len, context);
    FML_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128,
                "fml_attention_prefill: head_dim %u (need 32, 64 or 128)", head_dim);
    FML_REQUIRE(mode == FML_MATH_FP32 || mode == FML_MATH_TF32X3 || mode == FML_MATH_TF32,
                "fml_attention_prefill: unknown math mode %d", mode);
    const uint32_t ld = heads * head_dim;
    const uint64_t seq_stride = (uint64_t)heads * context * head_dim;
    cudaStream_t st = as_stream(stream);
    if (mode != FML_MATH_FP32)
    {
        const int rc = launch_prefill_attention_tc(q, ld, kcache, vcache, seq_stride, context, out, ld, batch, heads,
                                                   prompt_len, head_dim, scale, mode == FML_MATH_TF32X3, st);
        if (rc != FML_ERR_UNSUPPORTED) return rc;
    }
    return launch_prefill_attention(q, ld, kcache, vcache, seq_stride, context, out, ld, batch, heads, prompt_len,
                                    head_dim, scale, st);
}
