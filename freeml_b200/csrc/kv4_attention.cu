// Attention of one query row per sequence over the 4-bit paged cache.
//
// Mathematics.  A cached value is minimum + code * scale of its group of 32
// columns, so for a query head q and key k
//   q . k = sum_g scale_g (sum_{d in g} q_d code_d) + minimum_g (sum_{d in g} q_d)
// and for the output column d of group g
//   sum_k p_k v_kd = sum_k (p_k scale_kg) code_kd + sum_k p_k minimum_kg.
// The sums over codes are products of 16-bit halves with fp32 accumulators
// (mma.sync): the codes are the 16-row operand, 16 keys or 16 columns, and 8
// query heads the 8 columns of the other.  The keys' pairs are an operand as
// they lie (16-bit types): row (scale_0, minimum_0, scale_1, ...) times (0, sum_0
// q, 0, ...).
//
// Precision.  q is scaled by a power of two into the halves' range, and p is
// taken against a running maximum, 2^4 over which it moves; p enters the output and
// its sum alike, so that the maximum cancels.  p times a scale is moved to the top
// of the halves' range by a power of two of its own group of 32 columns (by one for
// all, groups of a thousandth beside ones near fp16's limit were 1e-3 off).  Each 16
// keys' products are a sum of their own, added in fp32.  What an output is off by
// goes by the largest values of its group: one near 0 is minimum + code scale too.
//   fp32: q and p go in as two halves each, hi and the remainder lo (22 bits);
//   codes are made normal halves about their middle (code - 8 for keys, - 7.5
//   for values), or the sums over codes would be large numbers that the minima's
//   sums take away again, and a group's middle, minimum + 8 scale, is formed in
//   fp32 before it meets the query (64 sequences of up to 1600 keys: 2e-5 off;
//   centred, 9e-7; with the middles, 3e-7; with a range for each group, 2.5e-7,
//   the formula in plain fp32 4e-7).
//   16-bit types: q is a half exactly; a code needs one AND to be an operand,
//   because bits 0..3 (4..7) of a half ARE the number code * 2^-24 (2^-20).
//   Products of such small halves are exact to 2^-17 (2^-21) of 15 codes: enough
//   for scores; the values' codes all go in at 2^-20 (a shift more).  p goes in as
//   hi and lo all the same.
//
// Work.  What bounds it is the cache's bytes, and the instructions that unpack
// them.  The keys of all sequences are cut into segments of about equal
// length, one CTA each, so that ragged batches fill the GPU; a segment is
// found from the lengths on the device.  Each of the CTA's warps streams its
// own tiles (2560 bytes: 16, 32 or 64 keys) through a ring of cp.async stages,
// whole ones, of which a count says the keys that are the sequence's, and keeps its
// own running maximum, sum and output in registers.  Segments of a split sequence
// leave partial results, which a second kernel joins.  About 380 (fp32, head dim 64)
// and 455 (16 bit, 128) instructions per 16 keys keep 61 % and 59 % of the issue
// slots busy: 64 sequences of 1600 keys, 16 heads of 64, fp32, take 69 us on a B200
// (1.9 TB/s); 8 of up to 65537, 32 on 8 heads of 128, bf16, 92 us (3.0 TB/s).
#include <type_traits>

#include "f32x2.cuh"
#include "kv4.cuh"

namespace fml {
namespace {

constexpr int GQ = 8;       // query heads of a CTA (rows of the products' hi half)
constexpr int NW = 4;       // warps
constexpr int STAGES = 4;   // tiles in flight per warp
constexpr int TILE = 2560;  // bytes of a tile
constexpr uint32_t MIN_SEGMENT = 256;  // keys
// CTAs an SM holds: head dim 128 needs the registers of 3 (8 long sequences of
// grouped heads, before sums were kept outside the products: 80 us against 92 at 4
// with 128 registers a thread)
constexpr int ctas_per_sm(int head_dim) { return head_dim == 128 ? 3 : 4; }

template <typename T>
struct Kv4AttnArgs
{
    T* out;
    const T* q;
    uint32_t ldo, ldq;
    const unsigned char* pool;
    uint32_t batch;
    uint32_t group;     // query heads of a key/value head
    uint32_t heads;
    uint32_t segments;  // bound of the segments of one head
    uint32_t spread;    // segments that all keys of one head are cut into, about
    float scale;
    float* partial;     // [segments][kv_heads][chunks][GQ][HD + 2]
    uint2* where;       // [batch]: first segment, number of segments
    Kv4View c;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the same with zeros for accumulators
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1)
{
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// 2^x by the hardware approximation (relative error about 2^-22)
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }

// two floats as halves, and what the halves leave of them as halves
__device__ __forceinline__ void split2(float2 x, uint32_t* hi, uint32_t* lo)
{
    const __half2 h = __float22half2_rn(x);
    const float2 r = fma2(__half22float2(h), make_float2(-1.f, -1.f), x);
    *hi = half2_bits(h);
    *lo = half2_bits(__float22half2_rn(r));
}

__device__ __forceinline__ float low_half(uint32_t u) { return __low2float(bits_half2(u)); }

// Row n, columns 2 c, 2 c + 1 of an 8 x 8 matrix of halves -> of its transpose.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// N = 1, 2 or 4 consecutive words, aligned to as many
template <int N>
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[N])
{
    if constexpr (N == 4)
    {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
    else if constexpr (N == 2)
    {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[1] = v.y;
    }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}

// Two codes (bits 0..3, or 4..7, of a word's halves) as an operand.
template <bool FULL>
__device__ __forceinline__ uint32_t codes_low(uint32_t w)
{
    if constexpr (FULL)  // 1024 + code as a half, less 1032
        return half2_bits(__hsub2(bits_half2((w & 0x000f000fu) | 0x64006400u), bits_half2(0x64086408u)));
    return w & 0x000f000fu;
}
template <bool FULL>
__device__ __forceinline__ uint32_t codes_high(uint32_t w)
{
    if constexpr (FULL)  // 1024 + 16 code as a half, a sixteenth of it less 72
        return half2_bits(
            __hfma2(bits_half2((w & 0x00f000f0u) | 0x64006400u), bits_half2(0x2c002c00u), bits_half2(0xd480d480u)));
    return w & 0x00f000f0u;
}

// Two values' codes, bits 4..7 of a word's halves, as an operand: less 7.5, their
// middle, or times 2^-20 (not, as keys' codes, some times 2^-24: 2^-17 of a group's
// range is then lost, which values near zero, minimum and codes cancelling, show).
template <bool FULL>
__device__ __forceinline__ uint32_t value_codes(uint32_t w)
{
    if constexpr (FULL)
        return half2_bits(
            __hfma2(bits_half2((w & 0x00f000f0u) | 0x64006400u), bits_half2(0x2c002c00u), bits_half2(0xd478d478u)));
    return w & 0x00f000f0u;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// acc += a (hi + lo) f, the products' sum rounded into acc; f a power of two
__device__ __forceinline__ void add_products(float (&acc)[4], const uint32_t (&a)[4], const uint32_t (&hi)[2],
                                             const uint32_t (&lo)[2], float f)
{
    float d[4];
    mma_f16_zero(d, a[0], a[1], a[2], a[3], lo[0], lo[1]);
    mma_f16(d, a, hi[0], hi[1]);
#pragma unroll
    for (int x = 0; x < 4; ++x) acc[x] = fmaf(d[x], f, acc[x]);
}

struct Segment
{
    uint32_t b, index, of, first;  // entry, number among its `of` segments, its first segment's number
};

// Segment number `idx` of one head: entries in order, each cut into equal
// parts.  Called by every thread of the CTA; of = 0 where there is none.
template <typename T>
__device__ Segment find_segment(const Kv4AttnArgs<T>& a, uint32_t idx)
{
    constexpr int NT = 32 * NW;
    __shared__ uint32_t warp_s[NW];
    __shared__ Segment seg_s;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (tid == 0) seg_s.of = 0;
    const uint32_t per = (a.batch + NT - 1) / NT, b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    uint64_t keys = 0;
    uint32_t len0 = 0;
    for (uint32_t b = b0; b < b1; ++b)
    {
        const uint32_t n = kv4_len(a.c, kv4_slot(a.c, b));
        if (b == b0) len0 = n;
        keys += n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) keys += __shfl_xor_sync(FULL_MASK, keys, o);
    __shared__ uint64_t keys_s[NW];
    if (lane == 0) keys_s[warp] = keys;
    __syncthreads();
    keys = 0;
    for (int w = 0; w < NW; ++w) keys += keys_s[w];
    // at most keys / chunk + batch segments: the launch's bound
    const uint64_t fair = (keys + a.spread - 1) / a.spread;
    const uint32_t chunk = (uint32_t)(fair < MIN_SEGMENT ? MIN_SEGMENT : fair < (1u << 31) ? fair : 1u << 31);
    uint32_t mine = 0;
    for (uint32_t b = b0; b < b1; ++b)
    {
        const uint32_t n = b == b0 ? len0 : kv4_len(a.c, kv4_slot(a.c, b));
        mine += n ? (n + chunk - 1) / chunk : 1u;  // an empty sequence: one, to write its zeros
    }
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    uint32_t at = x - mine;
    for (uint32_t w = 0; w < warp; ++w) at += warp_s[w];
    if (idx >= at && idx < at + mine)
        for (uint32_t b = b0; b < b1; ++b)
        {
            const uint32_t n = b == b0 ? len0 : kv4_len(a.c, kv4_slot(a.c, b));
            const uint32_t of = n ? (n + chunk - 1) / chunk : 1u;
            if (idx < at + of)
            {
                seg_s = Segment{b, idx - at, of, at};
                break;
            }
            at += of;
        }
    __syncthreads();
    return seg_s;
}

template <typename T, int HD>
__global__ void __launch_bounds__(32 * NW, ctas_per_sm(HD)) kv4_attention_kernel(Kv4AttnArgs<T> a)
{
    using B = Kv4Block<HD>;
    constexpr int NG = B::NG;
    constexpr int NSUB = 4 / NG;          // 16-key subtiles of a tile
    constexpr int KEYS = 16 * NSUB;       // keys of a tile
    constexpr int KCODE = 0, KMETA = 1024, VMETA = 1280, VCODE = 1536;
    __shared__ __align__(16) unsigned char ring[NW][STAGES][TILE];
    __shared__ uint32_t live_s[NW][STAGES][NSUB];  // keys of a subtile that count
    __shared__ float ml_s[NW][GQ][2];
    static_assert(sizeof(float) * GQ * HD <= sizeof(ring[0]), "a warp's output fits its ring");

    const Segment sg = find_segment(a, blockIdx.x);
    if (sg.of == 0) return;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t n = lane >> 2, c = lane & 3u;  // the products' column / row, and quarter
    const uint32_t kvh = blockIdx.y, g0 = blockIdx.z * GQ, nq = min((uint32_t)GQ, a.group - g0);
    const uint32_t h0 = kvh * a.group + g0;
    const uint32_t slot = kv4_slot(a.c, sg.b), len = kv4_len(a.c, slot);
    // equal parts in whole tiles of the CTA's warps
    const uint32_t part = ((len + sg.of - 1) / sg.of + KEYS - 1) / KEYS * KEYS;
    const uint32_t begin = min(sg.index * part, len), end = min(begin + part, len);
    const uint32_t tiles = (end - begin + KEYS - 1) / KEYS;
    const uint32_t mine = tiles > warp ? (tiles - warp + NW - 1) / NW : 0u;
    const uint32_t page_size = 1u << a.c.page_shift, block = B::bytes(page_size);
    const int32_t* trow = a.c.table + (uint64_t)(slot == ~0u ? 0u : slot) * a.c.max_pages;

    // The subtile whose table entry this lane looks up; the entry of tile i,
    // -1 where there is none.
    const uint32_t key0 = begin + warp * KEYS;  // this warp's tile i starts at key0 + i * NW * KEYS
    auto page_of = [&](uint32_t i) {
        const uint32_t k0 = key0 + i * (NW * KEYS) + 16 * (lane % NSUB);
        int32_t p = -1;
        if (k0 < end) p = trow[k0 >> a.c.page_shift];
        return (uint32_t)p < a.c.pages ? p : -1;
    };
    // A lane's five 16-byte pieces of a tile: codes of keys and of values (the
    // first and the second KB half), and pairs.  Whole tiles are copied: what
    // lies past a sequence's end, or (page 0) in the place of a missing page,
    // is masked by the count of live keys, and codes are finite whatever they are.
    constexpr uint32_t CS = 1024 / NSUB, MS = 256 / NSUB;  // a subtile's bytes
    const uint32_t oc = 16 * lane, om = 16 * (lane & 15u);
    const uint32_t s0 = oc / CS, s1 = (oc + 512) / CS, sm = om / MS;  // the pieces' subtiles
    const uint32_t row_mask = page_size - 1u;
    const uint32_t page_bytes = a.c.kv_heads * block;
    const uint32_t v_at = B::v(page_size);
    const unsigned char* head = a.pool + (uint64_t)kvh * block;
    const unsigned char* c_src = head + oc % CS;
    const unsigned char* d_src = head + (oc + 512) % CS;
    const unsigned char* m_src = head + (lane < 16 ? B::kmeta(page_size) : B::vmeta(page_size)) + om % MS;
    const uint32_t ring0 = static_cast<uint32_t>(__cvta_generic_to_shared(ring[warp][0]));
    const uint32_t m_dst = (lane < 16 ? KMETA : VMETA) + om;
    // rows of four 16-byte chunks of value codes: spread over the banks for the reads of rows 2 c
    const uint32_t v_dst = VCODE + (NG == 4 ? oc ^ ((oc >> 7 & 3u) << 4) : oc);
    auto issue = [&](uint32_t i, int32_t page) {
        const uint32_t tile0 = key0 + i * (NW * KEYS);
        if (tile0 < end)
        {
            const uint32_t at = i % STAGES, dst = ring0 + at * TILE;
            if (lane < NSUB)
                live_s[warp][at][lane] = page < 0 ? 0u : min(16u, end - (tile0 + 16 * lane));
            const uint32_t safe = (uint32_t)max(page, 0);
            const uint32_t p0 = NSUB == 1 ? safe : __shfl_sync(FULL_MASK, safe, s0);
            const uint32_t p1 = NSUB == 1 ? safe : __shfl_sync(FULL_MASK, safe, s1);
            const uint32_t pm = NSUB == 1 ? safe : __shfl_sync(FULL_MASK, safe, sm);
            const unsigned char* c0 = c_src + ((uint64_t)p0 * page_bytes + ((tile0 + 16 * s0) & row_mask) * B::ROW);
            const unsigned char* c1 = d_src + ((uint64_t)p1 * page_bytes + ((tile0 + 16 * s1) & row_mask) * B::ROW);
            const unsigned char* cm = m_src + ((uint64_t)pm * page_bytes + ((tile0 + 16 * sm) & row_mask) * B::META);
            cp16(dst + KCODE + oc, c0);
            cp16(dst + KCODE + 512 + oc, c1);
            cp16(dst + v_dst, c0 + v_at);
            cp16(dst + 512 + v_dst, c1 + v_at);
            cp16(dst + m_dst, cm);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int32_t next = page_of(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
    {
        const int32_t p = next;
        next = page_of(i + 1);
        issue(i, p);
    }

    // ---- the query: row n, columns 32 g + 8 c .. + 7 of every group ----
    // codes 0, 4, 2, 6 of a word are one operand register's, 1, 5, 3, 7 the
    // other's; as small halves (not FULL) they lie at 2^-24 and at 2^-20
    constexpr bool FULL = std::is_same_v<T, float>;
    constexpr float LOW = FULL ? 1.f : 16.f;
    uint32_t qh[NG][2][2], ql[FULL ? NG : 1][2][2], ua[2];
    float qf, uf;
    float2 qsum[FULL ? NG : 1];  // fp32: sum q of a group, heads 2 c and 2 c + 1, as the scores take it
    {
        float x[NG][8], top = 0.f, sum = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                x[g][e] = n < nq ? to_f32(a.q[(uint64_t)sg.b * a.ldq + (h0 + n) * HD + 32 * g + 8 * c + e]) : 0.f;
                top = fmaxf(top, fabsf(x[g][e]));
            }
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 1));
        top = fmaxf(top, __shfl_xor_sync(FULL_MASK, top, 2));
        // |q| 2^-e in [0.5, 1): e from the exponent bits, kept where 2^-e and 2^e are normal
        int e = (int)(__float_as_uint(top) >> 23) - 126;
        e = e < -100 ? -100 : e > 100 ? 100 : e;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23), up = __uint_as_float((uint32_t)(127 + e) << 23);
        const float s2 = a.scale * 1.4426950408889634f;  // scores in log2 units
        qf = FULL ? s2 * up : s2 * up * 1048576.0f;
        uf = s2 * up * 64.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
        {
            float s = ((x[g][0] + x[g][1]) + (x[g][2] + x[g][3])) + ((x[g][4] + x[g][5]) + (x[g][6] + x[g][7]));
            s += __shfl_xor_sync(FULL_MASK, s, 1);
            s += __shfl_xor_sync(FULL_MASK, s, 2);
            if constexpr (FULL)
                qsum[g] = make_float2(s2 * __shfl_sync(FULL_MASK, s, 8 * c), s2 * __shfl_sync(FULL_MASK, s, 8 * c + 4));
            else if (c == (uint32_t)g) sum = s * down * 0.015625f;  // a quarter's pair is its group's
#pragma unroll
            for (int h = 0; h < 2; ++h)
            {
                uint32_t l0, l1;
                split2(make_float2(x[g][2 * h] * down * LOW, x[g][2 * h + 4] * down * LOW), &qh[g][h][0], &l0);
                split2(make_float2(x[g][2 * h + 1] * down, x[g][2 * h + 5] * down), &qh[g][h][1], &l1);
                if constexpr (FULL) ql[g][h][0] = l0, ql[g][h][1] = l1;
            }
        }
        split2(make_float2(0.f, sum), &ua[0], &ua[1]);  // times (scale, minimum) of group c
    }
    // the factors of heads 2 c, 2 c + 1, whose scores this thread has
    const float2 qf2 = make_float2(__shfl_sync(FULL_MASK, qf, 8 * c), __shfl_sync(FULL_MASK, qf, 8 * c + 4));
    const float2 uf2 = make_float2(__shfl_sync(FULL_MASK, uf, 8 * c), __shfl_sync(FULL_MASK, uf, 8 * c + 4));
    // heads past the group's last see no key
    const float2 none2 = make_float2(2 * c < nq ? 0.f : -INFINITY, 2 * c + 1 < nq ? 0.f : -INFINITY);

    griddep_launch_dependents();
    // of heads 2 c, 2 c + 1: the reference exponent, and this thread's share of the sum
    float ref[2] = {-INFINITY, -INFINITY}, base[2] = {0.f, 0.f}, edge[2] = {-INFINITY, -INFINITY};
    float2 l = make_float2(0.f, 0.f);
    float acc[NG][2][4];  // columns 32 g + 4 n + 2 i (+ 1: the upper two) of both heads
    float2 u2[NG];        // sum p minimum (FULL: minimum + 7.5 scale) over this thread's keys
    // e of each group, in a float's place: p scale stays below 2^(e - 126) and goes in 2^(141 - e) times
    // larger; at the least for p = 2^4 by the smallest scale
    constexpr uint32_t LEAST = 107u << 23;
    constexpr uint32_t DOWN = (uint32_t)((FULL ? -14 : 6) * (1 << 23));  // 2^(e - 141), of codes at 2^-20 2^(e - 121)
    uint32_t unit[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g)
    {
        u2[g] = make_float2(0.f, 0.f);
        unit[g] = LEAST;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[g][i][e] = 0.f;
    }

    for (uint32_t i = 0; i < mine; ++i)
    {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncwarp();
        {
            const int32_t p = next;
            next = page_of(i + STAGES);
            issue(i + STAGES - 1, p);  // into the slot that the previous iteration read
        }
        const unsigned char* t = ring[warp][i % STAGES];
#pragma unroll
        for (int sub = 0; sub < NSUB; ++sub)
        {
            const uint32_t live = live_s[warp][i % STAGES][sub];
            // ---- scores of keys n and n + 8, heads 2 c and 2 c + 1 ----
            float2 s[2];
            {
                uint32_t w[2][NG], km[2][NG];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                {
                    load_words<NG>(t + KCODE + (16 * sub + 8 * k + n) * B::ROW + c * (4 * NG), w[k]);
                    load_words<NG>(t + KMETA + (16 * sub + 8 * k + n) * B::META, km[k]);
                }
                float du[4];
                if constexpr (!FULL)
                {
                    // the pair of group c; no such group: zeros (the query's side is 0 too, but 0 * NaN is not)
                    uint32_t pair[2] = {0u, 0u};
                    if (c < NG)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            pair[k] =
                                *reinterpret_cast<const uint32_t*>(t + KMETA + (16 * sub + 8 * k + n) * B::META + 4 * c);
                    mma_f16_zero(du, pair[0], pair[1], pair[0], pair[1], ua[0], ua[1]);  // hi, then lo, along k
                }
                float2 tt[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int g = 0; g < NG; ++g)
                {
                    const uint32_t r0 = w[0][g] >> 8, r1 = w[1][g] >> 8;
                    const uint32_t a0[4] = {codes_low<FULL>(w[0][g]), codes_low<FULL>(w[1][g]), codes_high<FULL>(w[0][g]),
                                            codes_high<FULL>(w[1][g])};
                    const uint32_t a1[4] = {codes_low<FULL>(r0), codes_low<FULL>(r1), codes_high<FULL>(r0),
                                            codes_high<FULL>(r1)};
                    float d[4];
                    if constexpr (FULL)  // the small products first
                    {
                        mma_f16_zero(d, a0[0], a0[1], a0[2], a0[3], ql[g][0][0], ql[g][0][1]);
                        mma_f16(d, a1, ql[g][1][0], ql[g][1][1]);
                        mma_f16(d, a0, qh[g][0][0], qh[g][0][1]);
                    }
                    else mma_f16_zero(d, a0[0], a0[1], a0[2], a0[3], qh[g][0][0], qh[g][0][1]);
                    mma_f16(d, a1, qh[g][1][0], qh[g][1][1]);
                    const float k0 = low_half(km[0][g]), k1 = low_half(km[1][g]);
                    tt[0] = fma2(make_float2(k0, k0), make_float2(d[0], d[1]), tt[0]);
                    tt[1] = fma2(make_float2(k1, k1), make_float2(d[2], d[3]), tt[1]);
                }
                if constexpr (FULL)
                {
                    // the groups' middles, minimum + 8 scale: the two would cancel in a product
                    float2 mid[2] = {none2, none2};
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                        {
                            const float2 v = __half22float2(bits_half2(km[k][g]));  // scale, minimum
                            const float m = fmaf(8.f, v.x, v.y);
                            mid[k] = fma2(make_float2(m, m), qsum[g], mid[k]);
                        }
                    s[0] = fma2(qf2, tt[0], mid[0]);
                    s[1] = fma2(qf2, tt[1], mid[1]);
                }
                else
                {
                    s[0] = fma2(qf2, tt[0], fma2(uf2, make_float2(du[0], du[1]), none2));
                    s[1] = fma2(qf2, tt[1], fma2(uf2, make_float2(du[2], du[3]), none2));
                }
            }
            // ---- the values' pairs of keys n, n + 8 ----
            uint32_t vm[2][NG];
#pragma unroll
            for (int k = 0; k < 2; ++k) load_words<NG>(t + VMETA + (16 * sub + 8 * k + n) * B::META, vm[k]);
            if (live < 16)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    if (n + 8 * k >= live)
                    {
                        s[k] = make_float2(-INFINITY, -INFINITY);
#pragma unroll
                        for (int g = 0; g < NG; ++g) vm[k][g] = 0u;
                    }
            // the scales as their group's power of two leaves them (negative where a constant group's
            // minimum was rounded up past it): with p of at most 2^4 below 2^15, or it is chosen again
            float sc[2][NG], most = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g)
            {
                const float up = __uint_as_float(0x86000000u - unit[g]);
#pragma unroll
                for (int k = 0; k < 2; ++k) sc[k][g] = low_half(vm[k][g]) * up;
                most = fmaxf(most, fmaxf(fabsf(sc[0][g]), fabsf(sc[1][g])));
            }
            const float2 top2 = make_float2(fmaxf(s[0].x, s[1].x), fmaxf(s[0].y, s[1].y));
            const bool over = most >= 2048.f, risen = top2.x > edge[0] || top2.y > edge[1];
            bool moved = false, wide = false;
            if (__any_sync(FULL_MASK, over || risen))
            {
                moved = __any_sync(FULL_MASK, risen);
                wide = __any_sync(FULL_MASK, over);
                float corr[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                {
                    float mx = h ? top2.y : top2.x;
                    mx = fmaxf(mx, __shfl_xor_sync(FULL_MASK, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(FULL_MASK, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(FULL_MASK, mx, 16));
                    // the reference moves only when a p would pass 2^4
                    const bool need = mx > ref[h] + 4.f;
                    const float fresh = need ? mx : ref[h];
                    corr[h] = need ? ex2(ref[h] - fresh) : 1.f;
                    ref[h] = fresh;
                    base[h] = fresh == -INFINITY ? 0.f : fresh;  // no key yet: 2^(-inf - 0) = 0
                    edge[h] = fresh + 4.f;
                }
                l.x *= corr[0];
                l.y *= corr[1];
#pragma unroll
                for (int g = 0; g < NG; ++g)
                {
                    u2[g].x *= corr[0];
                    u2[g].y *= corr[1];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) acc[g][j][x] *= corr[x & 1];
                }
            }
            float2 p[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) p[k] = make_float2(ex2(s[k].x - base[0]), ex2(s[k].y - base[1]));
            l.x += p[0].x + p[1].x;
            l.y += p[0].y + p[1].y;

            if (moved || wide)
            {
                // their groups' exponents again: what the subtile's keys ask for, and, while the maximum
                // stays, the earlier ones', with room for scales 2^6 larger.  A key that hardly counts asks
                // for its product alone.
                const float pm[2] = {fmaxf(p[0].x, p[0].y), fmaxf(p[1].x, p[1].y)};
#pragma unroll
                for (int g = 0; g < NG; ++g)
                {
                    float big = __uint_as_float(LEAST);
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        big = fmaxf(big, fabsf(low_half(vm[k][g])) * (pm[k] >= 0x1p-12f ? 16.f : pm[k]));
                    const uint32_t field = (__reduce_max_sync(FULL_MASK, __float_as_uint(big)) & 0x7f800000u) + (6u << 23);
                    const uint32_t to = moved ? field : max(unit[g], field);
                    const float up = __uint_as_float(0x86000000u - to);
                    unit[g] = to;
#pragma unroll
                    for (int k = 0; k < 2; ++k) sc[k][g] = low_half(vm[k][g]) * up;
                }
            }

            // ---- output: codes of columns 32 g + 4 n + j of keys 2 c, 2 c + 1, 2 c + 8, 2 c + 9 ----
            uint32_t vw[4][(NG + 1) / 2];
#pragma unroll
            for (int k = 0; k < 4; ++k)
            {
                const uint32_t key = 16 * sub + 2 * c + (k & 1) + 8 * (k >> 1);
                if constexpr (NG == 4)  // the copy put chunk x of a row at x ^ c
                {
                    const uint2 v =
                        *reinterpret_cast<const uint2*>(t + VCODE + key * B::ROW + ((n >> 1) ^ c) * 16 + (n & 1) * 8);
                    vw[k][0] = v.x, vw[k][1] = v.y;
                }
                else if constexpr (NG == 2)
                    vw[k][0] = *reinterpret_cast<const uint32_t*>(t + VCODE + key * B::ROW + 4 * n);
                else vw[k][0] = *reinterpret_cast<const uint16_t*>(t + VCODE + key * B::ROW + 2 * n);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
            {
                const uint32_t sel = (g & 1) ? 0x7632 : 0x5410;
                const uint32_t z0 = __byte_perm(vw[0][g / 2], vw[1][g / 2], sel);
                const uint32_t z1 = __byte_perm(vw[2][g / 2], vw[3][g / 2], sel);
                // fp32: about 7.5, since what the codes' mean is off their middle stays in the sums over
                // the keys until u2 takes it away again (two shifts more than about 8)
                const uint32_t r0 = z0 >> 8, r1 = z1 >> 8;
                const uint32_t a0[4] = {value_codes<FULL>(z0 << 4), value_codes<FULL>(z0), value_codes<FULL>(z1 << 4),
                                        value_codes<FULL>(z1)};
                const uint32_t a1[4] = {value_codes<FULL>(z0 >> 4), value_codes<FULL>(r0), value_codes<FULL>(z1 >> 4),
                                        value_codes<FULL>(r1)};
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)
                {
                    const float2 v = __half22float2(bits_half2(vm[k][g]));  // scale, minimum
                    split2(mul2(p[k], make_float2(sc[k][g], sc[k][g])), &hi[k], &lo[k]);
                    hi[k] = transpose8(hi[k]);
                    lo[k] = transpose8(lo[k]);
                    const float mid = FULL ? fmaf(7.5f, v.x, v.y) : v.y;
                    u2[g] = fma2(p[k], make_float2(mid, mid), u2[g]);
                }
                // the tensor cores' running sums are cut, not rounded: sums of many keys are kept outside
                // them (kept there, fp16 outputs over 30,000 keys of about equal weight, where the values'
                // mean is what is left of the codes', were 1.2e-3 off, so 2e-4)
                const float down = __uint_as_float(unit[g] + DOWN);
                add_products(acc[g][0], a0, hi, lo, down);
                add_products(acc[g][1], a1, hi, lo, down);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warps' results ----
#pragma unroll
    for (int o = 4; o < 32; o <<= 1)
    {
        l.x += __shfl_xor_sync(FULL_MASK, l.x, o);
        l.y += __shfl_xor_sync(FULL_MASK, l.y, o);
    }
    __syncthreads();  // the ring is free
    float* mine_o = reinterpret_cast<float*>(ring[warp]);
#pragma unroll
    for (int g = 0; g < NG; ++g)
    {
        float2 u = u2[g];
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
        {
            u.x += __shfl_xor_sync(FULL_MASK, u.x, o);
            u.y += __shfl_xor_sync(FULL_MASK, u.y, o);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
        {
            const float v = h ? u.y : u.x;
            const float4 o =
                make_float4(acc[g][0][h] + v, acc[g][0][h + 2] + v, acc[g][1][h] + v, acc[g][1][h + 2] + v);
            *reinterpret_cast<float4*>(mine_o + (2 * c + h) * HD + 32 * g + 4 * n) = o;
        }
    }
    if (n == 0)
    {
        ml_s[warp][2 * c][0] = ref[0];
        ml_s[warp][2 * c][1] = l.x;
        ml_s[warp][2 * c + 1][0] = ref[1];
        ml_s[warp][2 * c + 1][1] = l.y;
    }
    __syncthreads();
    const bool whole = sg.of == 1;
    if (!whole && threadIdx.x == 0 && sg.index == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        a.where[sg.b] = make_uint2(sg.first, sg.of);
    if (whole && a.where && threadIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) a.where[sg.b] = make_uint2(0u, 1u);
    for (uint32_t x = threadIdx.x; x < nq * HD; x += 32 * NW)
    {
        const uint32_t r = x / HD, d = x % HD;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, ml_s[w][r][0]);
        const float base = top == -INFINITY ? 0.f : top;
        float sum = 0.f, o = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w)
        {
            const float f = ex2(ml_s[w][r][0] - base);
            sum = fmaf(ml_s[w][r][1], f, sum);
            o = fmaf(reinterpret_cast<const float*>(ring[w])[r * HD + d], f, o);
        }
        if (whole)
            a.out[(uint64_t)sg.b * a.ldo + (h0 + r) * HD + d] = from_f32<T>(sum == 0.f ? 0.f : o / sum);
        else
        {
            float* dst = a.partial +
                         ((((uint64_t)blockIdx.x * a.c.kv_heads + kvh) * gridDim.z + blockIdx.z) * GQ + r) * (HD + 2);
            dst[2 + d] = o;
            if (d == 0)
            {
                dst[0] = top;
                dst[1] = sum;
            }
        }
    }
}

// Joins the segments of split sequences: one CTA per (entry, query head), whose
// warps take the segments in turn (a warp alone waits for one segment after
// another: 10 us for 50 of them, against 3).
template <typename T, int HD>
__global__ void __launch_bounds__(32 * NW) kv4_join_kernel(Kv4AttnArgs<T> a, uint32_t chunks)
{
    constexpr int E = HD / 32;
    __shared__ float sum_s[NW], o_s[NW][HD];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, kvh = h / a.group, g = h % a.group;
    griddep_wait();
    const uint2 at = a.where[b];
    if (at.y <= 1) return;
    const uint64_t step = (uint64_t)a.c.kv_heads * chunks * GQ * (HD + 2);
    const float* p = a.partial + (uint64_t)at.x * step + (((uint64_t)kvh * chunks + g / GQ) * GQ + g % GQ) * (HD + 2);
    float top = -INFINITY;
    for (uint32_t s = lane; s < at.y; s += 32) top = fmaxf(top, p[s * step]);
    top = warp_max(top);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
    for (uint32_t s = warp; s < at.y; s += NW)
    {
        const float* r = p + s * step;
        const float f = ex2(r[0] - base);
        sum = fmaf(r[1], f, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(r[2 + 32 * e + lane], f, o[e]);
    }
    if (lane == 0) sum_s[warp] = sum;
#pragma unroll
    for (int e = 0; e < E; ++e) o_s[warp][32 * e + lane] = o[e];
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += sum_s[w];
    for (uint32_t d = threadIdx.x; d < HD; d += 32 * NW)
    {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) x += o_s[w][d];
        a.out[(uint64_t)b * a.ldo + h * HD + d] = from_f32<T>(sum == 0.f ? 0.f : x / sum);
    }
}

// Segments that one head's keys are cut into, about, and their bound.
struct Split
{
    uint32_t spread, segments, chunks;
    bool split;  // whether a sequence may be cut at all
};

Split plan(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_pages,
           uint32_t page_size)
{
    Split s;
    s.chunks = (heads / kv_heads + GQ - 1) / GQ;
    const uint64_t per_head = (uint64_t)kv_heads * s.chunks;
    // The CTAs of one wave, less one for each sequence's part-full segment,
    // where that leaves half of them.
    const uint64_t wave = (148u * ctas_per_sm((int)head_dim) + per_head - 1) / per_head;
    const uint64_t spread = wave > 2ull * batch ? wave - batch : (wave + 1) / 2;
    s.spread = (uint32_t)(spread < 1 ? 1 : spread);
    const uint64_t cap = (uint64_t)max_pages * page_size;
    const uint64_t most = batch * (cap <= MIN_SEGMENT ? 1 : (cap + MIN_SEGMENT - 1) / MIN_SEGMENT);
    const uint64_t bound = (uint64_t)s.spread + batch;
    s.segments = (uint32_t)(bound < most ? bound : most);
    s.split = cap > MIN_SEGMENT;
    return s;
}

size_t where_bytes(uint32_t batch) { return ((size_t)batch * sizeof(uint2) + 15) / 16 * 16; }

template <typename T, int HD>
int launch(const Kv4AttnArgs<T>& a, const Split& s, cudaStream_t st)
{
    kv4_attention_kernel<T, HD><<<dim3(s.segments, a.c.kv_heads, s.chunks), 32 * NW, 0, st>>>(a);
    FML_LAUNCH_CHECK();
    if (!s.split) return FML_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.batch * a.heads);
    cfg.blockDim = dim3(32 * NW);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    FML_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, HD>, a, s.chunks));
    FML_LAUNCH_CHECK();
    return FML_OK;
}

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" {

size_t fml_attention_kv4_workspace_bytes(uint32_t batch, uint32_t heads, uint32_t kv_heads, uint32_t head_dim,
                                         uint32_t max_pages, uint32_t page_size)
{
    if (batch == 0 || kv_heads == 0 || heads < kv_heads) return 0;
    const Split s = plan(batch, heads, kv_heads, head_dim, max_pages, page_size);
    if (!s.split) return 0;
    return where_bytes(batch) + (size_t)s.segments * kv_heads * s.chunks * GQ * (head_dim + 2) * sizeof(float);
}

int fml_attention_kv4(void* out, const void* q, int type, uint32_t ldo, uint32_t ldq, const void* pool,
                      const int32_t* table, const uint32_t* lens, const uint32_t* slot_ids, uint32_t batch,
                      uint32_t pages, uint32_t slots, uint32_t max_pages, uint32_t page_size, uint32_t heads,
                      uint32_t kv_heads, uint32_t head_dim, float scale, void* workspace, size_t workspace_bytes,
                      fml_stream_t stream)
{
    if (batch == 0) return FML_OK;
    FML_REQUIRE(out && q && pool && table && lens, "fml_attention_kv4: null pointer");
    FML_REQUIRE(aligned16(pool), "fml_attention_kv4: the pool must be 16-byte aligned");
    FML_REQUIRE(type == FML_TYPE_FP32 || type == FML_TYPE_FP16 || type == FML_TYPE_BF16,
                "fml_attention_kv4: unknown type %d", type);
    FML_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128,
                "fml_attention_kv4: head_dim %u (need 32, 64 or 128)", head_dim);
    FML_REQUIRE(kv4_page_shift(page_size) && (uint64_t)max_pages * page_size < (1ull << 31),
                "fml_attention_kv4: %u pages of %u rows a sequence", max_pages, page_size);
    FML_REQUIRE(pages >= 1 && pages < (1u << 31) && slots >= 1, "fml_attention_kv4: %u pages, %u slots", pages, slots);
    FML_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0,
                "fml_attention_kv4: %u query heads over %u key/value heads", heads, kv_heads);
    FML_REQUIRE((uint64_t)heads * head_dim <= ldq && (uint64_t)heads * head_dim <= ldo,
                "fml_attention_kv4: rows of %u heads of %u, strides %u and %u", heads, head_dim, ldq, ldo);
    FML_REQUIRE((uint64_t)kv_heads * fml_kv4_block_bytes(head_dim, page_size) < (1ull << 32),
                "fml_attention_kv4: pages of %u heads", kv_heads);
    FML_REQUIRE((uint64_t)batch * heads < (1ull << 31), "fml_attention_kv4: batch %u of %u heads", batch, heads);
    const Split s = plan(batch, heads, kv_heads, head_dim, max_pages, page_size);
    FML_REQUIRE(kv_heads <= 65535u && s.chunks <= 65535u, "fml_attention_kv4: %u heads", heads);
    const size_t need = fml_attention_kv4_workspace_bytes(batch, heads, kv_heads, head_dim, max_pages, page_size);
    FML_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
                "fml_attention_kv4: the workspace needs %zu bytes, 16-byte aligned", need);
    const Kv4View c{table, lens, slot_ids, pages, slots, max_pages, kv4_page_shift(page_size), kv_heads};
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const Kv4AttnArgs<T> a{static_cast<T*>(out),
                               static_cast<const T*>(q),
                               ldo,
                               ldq,
                               static_cast<const unsigned char*>(pool),
                               batch,
                               heads / kv_heads,
                               heads,
                               s.segments,
                               s.spread,
                               scale,
                               s.split ? reinterpret_cast<float*>(ws + where_bytes(batch)) : nullptr,
                               s.split ? reinterpret_cast<uint2*>(ws) : nullptr,
                               c};
        if (head_dim == 32) return launch<T, 32>(a, s, as_stream(stream));
        if (head_dim == 64) return launch<T, 64>(a, s, as_stream(stream));
        return launch<T, 128>(a, s, as_stream(stream));
    };
    if (type == FML_TYPE_FP32) return go(static_cast<float*>(nullptr));
    if (type == FML_TYPE_FP16) return go(static_cast<__half*>(nullptr));
    return go(static_cast<__nv_bfloat16*>(nullptr));
}

}  // extern "C"
