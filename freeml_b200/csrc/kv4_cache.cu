// The 4-bit paged key/value cache: rows written to it and read back, and the
// page operations (reserve, fork, free, compact).
//
// Rows.  A thread has eight consecutive columns of a key and of the value row,
// four neighbouring threads a group of 32: the group's extremes are two
// shuffles, and the eight key codes are one word.  A CTA takes a run of tokens;
// its first threads find each token's sequence (a binary search in the starts),
// page and row once for all heads.  Bound by the quantisation's instructions
// when writing (67 % of issue slots) and by the rows' bytes when reading: 10,152
// tokens of 8 heads of 128, bf16 in and fp32 out, take 26 and 28 us on a B200.
// (Four columns a thread, each thread finding its row's place: 84 us for both.)
//
// Pages.  Reference counts, tables and lengths are small integers; one CTA
// settles them (block scans over the counts, in page order, so that the lowest
// free page is always the next one; 7 us for 2600 pages, most of it the scans'
// barriers), and a second kernel moves the pages' bytes with the whole GPU: 104 MB
// of moved pages in 35 us, 5.9 TB/s read and written.
#include <type_traits>

#include "kv4.cuh"

namespace fml {
namespace {

constexpr float LIMIT = 65504.0f;  // fp16's largest value: pairs stay finite

template <typename T>
struct RowArgs
{
    unsigned char* pool;
    T* k;
    T* v;
    const uint32_t* starts;
    const uint32_t* kept;  // rows of a slot before kept[slot] are not written; null: all may be
    uint32_t batch, rows, ldk, ldv, tokens;  // tokens: rows of a CTA
    Kv4View c;
};

constexpr uint32_t MAX_TOKENS = 16;

// Where new row r lies: the offset of its page in the pool (head 0's block)
// and its row within the page; false where it has no place.
__device__ bool find_row(const Kv4View& c, const uint32_t* starts, const uint32_t* kept, uint32_t batch, uint32_t r,
                         uint64_t block_bytes, uint64_t* at, uint32_t* row)
{
    uint32_t lo = 0, hi = batch;  // the last entry whose start is at most r
    while (hi - lo > 1)
    {
        const uint32_t mid = (lo + hi) >> 1;
        if (starts[mid] <= r) lo = mid;
        else hi = mid;
    }
    const uint32_t end = starts[lo + 1];
    if (r < starts[lo] || r >= end) return false;
    const uint32_t slot = kv4_slot(c, lo), len = kv4_len(c, slot);
    if (end - r > len) return false;
    const uint32_t pos = len - (end - r);
    if (kept && pos < kept[slot]) return false;
    const int32_t page = c.table[(uint64_t)slot * c.max_pages + (pos >> c.page_shift)];
    if (page < 0 || (uint32_t)page >= c.pages) return false;
    *at = (uint64_t)page * c.kv_heads * block_bytes;
    *row = pos & ((1u << c.page_shift) - 1u);
    return true;
}

// Eight values of a group as codes; the pair goes to every thread of the four.
__device__ __forceinline__ uint32_t quantise8(float (&x)[8], __half2* pair)
{
    bool nan = false;
    float lo = LIMIT, hi = -LIMIT;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        nan |= x[i] != x[i];
        x[i] = fminf(fmaxf(x[i], -LIMIT), LIMIT);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
    {
        lo = fminf(lo, __shfl_xor_sync(FULL_MASK, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(FULL_MASK, hi, o));
    }
    const uint32_t nans = __ballot_sync(FULL_MASK, nan);
    nan = (nans >> (threadIdx.x & 28u) & 15u) != 0;
    const __half mn = __float2half_rn(lo);
    const float fm = __half2float(mn);
    const __half sc = __float2half_rn(__fmul_rn(hi - fm, 1.0f / 15.0f));
    const float fs = __half2float(sc);
    const float inv = fs == 0.0f ? 0.0f : __frcp_rn(fs);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
    {
        // round to nearest, ties to even, clamped: as a whole number in the low bits
        const float c = fminf(fmaxf(__fmul_rn(x[i] - fm, inv), 0.0f), 15.0f);
        codes |= (__float_as_uint(c + 12582912.0f) & 15u) << (4 * i);
    }
    const __half bad = __ushort_as_half(0x7fff);
    *pair = nan ? __halves2half2(bad, bad) : __halves2half2(sc, mn);
    return nan ? 0u : codes;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8])
{
    if constexpr (VEC)
    {
        union
        {
            uint4 u[sizeof(T) / 2];
            T e[8];
        } q;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) q.u[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(q.e[i]);
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[8])
{
    if constexpr (VEC)
    {
        union
        {
            uint4 u[sizeof(T) / 2];
            T e[8];
        } q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q.e[i] = from_f32<T>(x[i]);
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = q.u[i];
    }
    else
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_f32<T>(x[i]);
    }
}

// READ false: rows of k and v become cache rows; true: the reverse.
template <typename T, int HD, bool VEC, bool READ>
__global__ void __launch_bounds__(256) kv4_rows_kernel(RowArgs<T> a)
{
    using B = Kv4Block<HD>;
    constexpr int NG = B::NG;
    constexpr uint32_t UNITS = HD / 8;  // threads of a row
    __shared__ uint64_t at_s[MAX_TOKENS];
    __shared__ uint32_t row_s[MAX_TOKENS];
    const uint32_t page_size = 1u << a.c.page_shift, block = B::bytes(page_size);
    const uint32_t r0 = blockIdx.x * a.tokens;
    const uint32_t n = min(a.tokens, a.rows - r0);
    const uint32_t per_token = a.c.kv_heads * UNITS, total = n * per_token;
    // the values of the first pass are on their way while the rows are found
    float x[8], y[8];
    auto fetch = [&](uint32_t i) {
        const uint32_t u = i < total ? i : 0u, tok = u / per_token, col = (u - tok * per_token) * 8;
        load8<T, VEC>(a.k + (uint64_t)(r0 + tok) * a.ldk + col, x);
        load8<T, VEC>(a.v + (uint64_t)(r0 + tok) * a.ldv + col, y);
    };
    if constexpr (!READ) fetch(blockIdx.y * 256 + threadIdx.x);
    if (threadIdx.x < n)
    {
        uint64_t at = 0;
        uint32_t row = 0;
        const bool ok = find_row(a.c, a.starts, a.kept, a.batch, r0 + threadIdx.x, block, &at, &row);
        at_s[threadIdx.x] = at;
        row_s[threadIdx.x] = ok ? row : ~0u;
    }
    __syncthreads();
    for (uint32_t i0 = blockIdx.y * 256; i0 < total; i0 += gridDim.y * 256)
    {
        const uint32_t i = i0 + threadIdx.x, u = i < total ? i : 0u;
        const uint32_t tok = u / per_token, hu = u - tok * per_token;
        const uint32_t head = hu / UNITS, lane = hu % UNITS;
        const uint32_t row = row_s[tok];
        const bool live = i < total && row != ~0u;
        const uint32_t col = head * HD + 8 * lane;
        unsigned char* blk = a.pool + at_s[tok] + (uint64_t)head * block;
        // columns 32 g + 8 c ..: key word c * NG + g, value units 2 c * NG + g and (2 c + 1) * NG + g
        const uint32_t g = lane / 4, c = lane & 3u, r = live ? row : 0u;
        uint32_t* kw = reinterpret_cast<uint32_t*>(blk + r * B::ROW) + c * NG + g;
        __half2* kp = reinterpret_cast<__half2*>(blk + B::kmeta(page_size) + r * B::META) + g;
        uint16_t* vu = reinterpret_cast<uint16_t*>(blk + B::v(page_size) + r * B::ROW) + 2 * c * NG + g;
        __half2* vp = reinterpret_cast<__half2*>(blk + B::vmeta(page_size) + r * B::META) + g;
        if constexpr (READ)
        {
            if (live)
            {
                const uint32_t kc = *kw, vc = vu[0] | (uint32_t)vu[NG] << 16;
                const float2 km = __half22float2(*kp), vm = __half22float2(*vp);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                {
                    x[e] = fmaf((float)((kc >> (4 * e)) & 15u), km.x, km.y);
                    y[e] = fmaf((float)((vc >> (4 * e)) & 15u), vm.x, vm.y);
                }
                store8<T, VEC>(a.k + (uint64_t)(r0 + tok) * a.ldk + col, x);
                store8<T, VEC>(a.v + (uint64_t)(r0 + tok) * a.ldv + col, y);
            }
        }
        else
        {
            __half2 km, vm;
            const uint32_t kc = quantise8(x, &km), vc = quantise8(y, &vm);
            if (i0 + gridDim.y * 256 < total) fetch(i + gridDim.y * 256);
            if (live)
            {
                *kw = kc;
                vu[0] = (uint16_t)vc;
                vu[NG] = (uint16_t)(vc >> 16);
                if (c == 0)
                {
                    *kp = km;
                    *vp = vm;
                }
            }
        }
    }
}

template <typename T, int HD, bool READ>
int launch_rows(const RowArgs<T>& a, bool vec, cudaStream_t st)
{
    const uint32_t ctas = (a.rows + a.tokens - 1) / a.tokens;
    const uint64_t units = (uint64_t)(a.tokens < a.rows ? a.tokens : a.rows) * a.c.kv_heads * (HD / 8);
    const uint64_t parts = (units + 1023) / 1024;  // CTAs that share a run of tokens: up to four passes each
    const uint32_t y = (uint32_t)(parts < 65535u ? parts : 65535u);
    dim3 grid(ctas, y);
    if (vec) kv4_rows_kernel<T, HD, true, READ><<<grid, 256, 0, st>>>(a);
    else kv4_rows_kernel<T, HD, false, READ><<<grid, 256, 0, st>>>(a);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

int check_view(const char* who, const void* pool, const void* table, const void* lens, uint32_t pages, uint32_t slots,
               uint32_t max_pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim, uint32_t batch)
{
    FML_REQUIRE(pool && table && lens, "%s: null pointer", who);
    FML_REQUIRE(aligned16(pool), "%s: the pool must be 16-byte aligned", who);
    FML_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, "%s: head_dim %u (need 32, 64 or 128)", who,
                head_dim);
    FML_REQUIRE(kv4_page_shift(page_size), "%s: page_size %u (need 16, 32, 64 or 128)", who, page_size);
    FML_REQUIRE(pages >= 1 && pages < (1u << 31) && slots >= 1 && kv_heads >= 1, "%s: %u pages, %u slots, %u heads",
                who, pages, slots, kv_heads);
    FML_REQUIRE((uint64_t)max_pages * page_size < (1ull << 31), "%s: %u pages of %u rows a sequence", who, max_pages,
                page_size);
    FML_REQUIRE(batch < (1u << 31), "%s: batch %u", who, batch);
    return FML_OK;
}

template <bool READ>
int rows_entry(const char* who, void* pool, const int32_t* table, const uint32_t* lens, const uint32_t* slot_ids,
               const uint32_t* kept, void* k, void* v, int type, const uint32_t* starts, uint32_t batch, uint32_t rows,
               uint32_t ldk, uint32_t ldv, uint32_t pages, uint32_t slots, uint32_t max_pages, uint32_t page_size,
               uint32_t kv_heads, uint32_t head_dim, cudaStream_t st)
{
    if (batch == 0 || rows == 0) return FML_OK;
    FML_RC(check_view(who, pool, table, lens, pages, slots, max_pages, page_size, kv_heads, head_dim, batch));
    FML_REQUIRE(k && v && starts, "%s: null pointer", who);
    FML_REQUIRE(type == FML_TYPE_FP32 || type == FML_TYPE_FP16 || type == FML_TYPE_BF16, "%s: unknown type %d", who,
                type);
    FML_REQUIRE((uint64_t)kv_heads * head_dim <= ldk && (uint64_t)kv_heads * head_dim <= ldv,
                "%s: rows of %u heads of %u, strides %u and %u", who, kv_heads, head_dim, ldk, ldv);
    const bool vec = aligned16(k) && aligned16(v) && (ldk | ldv) * type_bytes(type) % 16 == 0;
    // tokens of a CTA: as many as leave every SM a few CTAs
    uint32_t tokens = rows / (148u * 16u);
    tokens = tokens < 1 ? 1 : tokens > MAX_TOKENS ? MAX_TOKENS : tokens;
    const Kv4View c{table, lens, slot_ids, pages, slots, max_pages, kv4_page_shift(page_size), kv_heads};
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        RowArgs<T> a{static_cast<unsigned char*>(pool), static_cast<T*>(k), static_cast<T*>(v), starts, kept, batch, rows,
                     ldk, ldv, tokens, c};
        if (head_dim == 32) return launch_rows<T, 32, READ>(a, vec, st);
        if (head_dim == 64) return launch_rows<T, 64, READ>(a, vec, st);
        return launch_rows<T, 128, READ>(a, vec, st);
    };
    if (type == FML_TYPE_FP32) return go(static_cast<float*>(nullptr));
    if (type == FML_TYPE_FP16) return go(static_cast<__half*>(nullptr));
    return go(static_cast<__nv_bfloat16*>(nullptr));
}

// ---- pages --------------------------------------------------------------------

constexpr uint32_t PT = 1024;  // threads of the CTA that settles the integers
constexpr uint32_t MAX_PAGES = 1u << 21;

// Exclusive sum of v over the CTA in thread order, and the total.
__device__ uint32_t block_exclusive(uint32_t v, uint32_t* total)
{
    __shared__ uint32_t warp_s[PT / 32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    __syncthreads();  // warp_s of the previous call has been read
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    uint32_t before = 0, all = 0;
    const uint32_t nw = blockDim.x >> 5;
    uint32_t s = lane < nw ? warp_s[lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint32_t y = __shfl_up_sync(FULL_MASK, s, o);
        if (lane >= (uint32_t)o) s += y;
    }
    all = __shfl_sync(FULL_MASK, s, 31);
    before = __shfl_sync(FULL_MASK, s, warp ? warp - 1 : 0);
    if (warp == 0) before = 0;
    *total = all;
    return before + x - v;
}

// The lowest `want` free pages, in order, into out; false (nothing of use in
// out) where there are fewer.  Four pages a thread and pass.
__device__ bool take_free(const int32_t* refs, uint32_t pages, uint32_t want, uint32_t* out)
{
    uint32_t have = 0;
    for (uint32_t p0 = 0; p0 < pages && have < want; p0 += 4 * PT)
    {
        uint32_t mine = 0, p = p0 + 4 * threadIdx.x;
        bool free4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            free4[i] = p + i < pages && refs[p + i] <= 0;
            mine += free4[i];
        }
        uint32_t total, at = have + block_exclusive(mine, &total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (free4[i])
            {
                if (at < want) out[at] = p + i;
                ++at;
            }
        have += total;
    }
    __syncthreads();
    return have >= want;
}

struct PageArgs
{
    int32_t* refs;
    int32_t* table;
    uint32_t* lens;
    uint32_t pages, slots, max_pages, page_shift;
    int32_t* status;
};

// Workspace words: [0] pairs to copy, [1] whether the call is carried out,
// then the lists.
constexpr uint32_t WS_HEAD = 16;

// reserve: need[i] pages for entry i; the claims (top bit of lens) find slots
// named twice.  kept (or null) [slots]: the lengths where the call is refused; no
// more than them where it is carried out.
__global__ void __launch_bounds__(PT) kv4_reserve_kernel(PageArgs a, const uint32_t* slot_ids, const uint32_t* counts,
                                                         uint32_t n, uint32_t* kept, uint32_t* ws)
{
    __shared__ uint32_t bad_s;
    uint32_t* need = ws + WS_HEAD;  // exclusive sums, n + 1
    uint32_t* fresh = need + n + 1;
    const uint32_t page = 1u << a.page_shift;
    if (threadIdx.x == 0) bad_s = 0;
    __syncthreads();
    uint32_t carry = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += PT)
    {
        const uint32_t i = i0 + threadIdx.x;
        uint32_t want = 0;
        if (i < n)
        {
            const uint32_t slot = slot_ids ? slot_ids[i] : i;
            if (slot >= a.slots) atomicOr(&bad_s, FML_KV4_BAD_SLOT);
            else
            {
                const uint32_t old = atomicOr(&a.lens[slot], 0x80000000u);
                if (old & 0x80000000u) atomicOr(&bad_s, FML_KV4_BAD_SLOT);
                else if ((uint64_t)old + counts[i] > (uint64_t)a.max_pages << a.page_shift)
                    atomicOr(&bad_s, FML_KV4_ROW_FULL);
                else
                    want = ((old + counts[i] + page - 1) >> a.page_shift) - ((old + page - 1) >> a.page_shift);
                if (want > a.pages)
                {
                    atomicOr(&bad_s, FML_KV4_NO_PAGES);
                    want = 0;
                }
            }
        }
        uint32_t total, at = block_exclusive(want, &total);  // at most PT * MAX_PAGES = 2^31
        if (i < n) need[i] = carry + at;
        carry = min(carry + total, 1u << 30);
    }
    __syncthreads();
    bool ok = bad_s == 0;
    __syncthreads();  // read by all before thread 0 may write it again
    if (ok && (carry > a.pages || !take_free(a.refs, a.pages, carry, fresh)))
    {
        ok = false;
        if (threadIdx.x == 0) bad_s = FML_KV4_NO_PAGES;
    }
    __syncthreads();
    if (ok)
    {
        for (uint32_t i = threadIdx.x; i < n; i += PT)
        {
            const uint32_t slot = slot_ids ? slot_ids[i] : i;
            const uint32_t old = a.lens[slot] & 0x7fffffffu, from = (old + page - 1) >> a.page_shift;
            const uint32_t end = i + 1 < n ? need[i + 1] : carry;
            for (uint32_t j = need[i]; j < end; ++j)
            {
                a.table[(uint64_t)slot * a.max_pages + from + (j - need[i])] = (int32_t)fresh[j];
                a.refs[fresh[j]] = 1;
            }
            a.lens[slot] = old + counts[i];
            if (kept) kept[slot] = min(kept[slot], old);
        }
        return;
    }
    // nothing changes: the claims are taken back
    for (uint32_t i = threadIdx.x; i < n; i += PT)
    {
        const uint32_t slot = slot_ids ? slot_ids[i] : i;
        if (slot >= a.slots) continue;
        const uint32_t old = atomicAnd(&a.lens[slot], 0x7fffffffu) & 0x7fffffffu;
        if (kept) kept[slot] = old;
    }
    if (threadIdx.x == 0) atomicOr(a.status, (int)bad_s);
}

// fork: settles lengths and pages; the next kernel copies tables and pages.
// Workspace lists: rows[n] (the parent's length), first[n] (exclusive sums of
// pages to copy), fresh[n].
__global__ void __launch_bounds__(PT) kv4_fork_kernel(PageArgs a, const uint32_t* parents, const uint32_t* children,
                                                      uint32_t n, uint32_t* ws)
{
    __shared__ uint32_t bad_s;
    uint32_t* rows = ws + WS_HEAD;
    uint32_t* src = rows + n;  // page to copy, or ~0
    uint32_t* dst = src + n;
    uint32_t* fresh = dst + n;
    const uint32_t page = 1u << a.page_shift;
    if (threadIdx.x == 0) bad_s = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n; i += PT)
    {
        const uint32_t p = parents[i], c = children[i];
        if (p >= a.slots || c >= a.slots) atomicOr(&bad_s, FML_KV4_BAD_SLOT);
        else rows[i] = min(a.lens[p], a.max_pages << a.page_shift);
    }
    __syncthreads();
    const bool slots_ok = bad_s == 0;
    __syncthreads();  // read by all before a claim may write it: all take the same side of what follows
    if (slots_ok)
    {
        // a child must be empty and named once: claim it
        uint32_t carry = 0;
        for (uint32_t i0 = 0; i0 < n; i0 += PT)
        {
            const uint32_t i = i0 + threadIdx.x;
            uint32_t want = 0;
            if (i < n)
            {
                const bool mine = atomicCAS(&a.lens[children[i]], 0u, ~0u) == 0u;
                if (!mine) atomicOr(&bad_s, FML_KV4_BAD_SLOT);
                const uint32_t full = rows[i] >> a.page_shift;
                int32_t from = -1;
                if (rows[i] & (page - 1u)) from = a.table[(uint64_t)parents[i] * a.max_pages + full];
                const bool copy = from >= 0 && (uint32_t)from < a.pages;
                src[i] = copy ? (uint32_t)from : ~0u;
                want = copy;
                dst[i] = mine;  // until the claims are settled
            }
            uint32_t total, at = block_exclusive(want, &total);
            if (i < n && want) fresh[n + i] = carry + at;  // its place among the fresh pages
            carry += total;
        }
        __syncthreads();
        bool ok = bad_s == 0;
        if (ok && !take_free(a.refs, a.pages, carry, fresh))
        {
            ok = false;
            if (threadIdx.x == 0) bad_s = FML_KV4_NO_PAGES;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += PT)
        {
            if (!ok)
            {
                if (dst[i]) a.lens[children[i]] = 0;
                continue;
            }
            a.lens[children[i]] = rows[i];
            dst[i] = ~0u;
            if (src[i] != ~0u)
            {
                dst[i] = fresh[fresh[n + i]];
                a.refs[dst[i]] = 1;
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0)
    {
        ws[0] = bad_s ? 0u : n;
        if (bad_s) atomicOr(a.status, (int)bad_s);
    }
}

// Copies page src[i] to dst[i] (~0: none) in every layer, for the pairs that
// the first kernel left; 16 KB a CTA and step.
__device__ void copy_pages(unsigned char* pool, uint32_t layers, uint64_t layer_stride, uint64_t page_bytes,
                           const uint32_t* src, const uint32_t* dst, uint32_t n)
{
    const uint64_t vecs = page_bytes / 16;
    const uint32_t steps = (uint32_t)((vecs + 1023) / 1024);
    const uint64_t total = (uint64_t)n * layers * steps;
    for (uint64_t w = blockIdx.x; w < total; w += gridDim.x)
    {
        const uint64_t pl = w / steps;
        const uint32_t step = (uint32_t)(w - pl * steps), i = (uint32_t)(pl / layers), l = (uint32_t)(pl % layers);
        if (src[i] == ~0u || dst[i] == ~0u) continue;
        const uint4* s = reinterpret_cast<const uint4*>(pool + l * layer_stride + src[i] * page_bytes);
        uint4* d = reinterpret_cast<uint4*>(pool + l * layer_stride + dst[i] * page_bytes);
        uint4 x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            const uint64_t j = (uint64_t)step * 1024 + e * 256 + threadIdx.x;
            if (j < vecs) x[e] = s[j];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
        {
            const uint64_t j = (uint64_t)step * 1024 + e * 256 + threadIdx.x;
            if (j < vecs) d[j] = x[e];
        }
    }
}

__global__ void __launch_bounds__(256) kv4_fork_copy_kernel(PageArgs a, unsigned char* pool, uint32_t layers,
                                                            uint64_t layer_stride, uint64_t page_bytes,
                                                            const uint32_t* parents, const uint32_t* children,
                                                            uint32_t n, const uint32_t* ws)
{
    const uint32_t pairs = ws[0];
    const uint32_t* rows = ws + WS_HEAD;
    const uint32_t* src = rows + n;
    const uint32_t* dst = src + n;
    if (pairs == 0) return;
    // the children's tables, and the counts of the shared pages
    const uint64_t cells = (uint64_t)pairs * a.max_pages;
    for (uint64_t x = blockIdx.x * 256ull + threadIdx.x; x < cells; x += gridDim.x * 256ull)
    {
        const uint32_t i = (uint32_t)(x / a.max_pages), col = (uint32_t)(x % a.max_pages);
        const uint32_t full = rows[i] >> a.page_shift;
        int32_t p = -1;
        if (col < full)
        {
            p = a.table[(uint64_t)parents[i] * a.max_pages + col];
            if (p >= 0 && (uint32_t)p < a.pages) atomicAdd(&a.refs[p], 1);
        }
        else if (col == full && dst[i] != ~0u) p = (int32_t)dst[i];
        a.table[(uint64_t)children[i] * a.max_pages + col] = p;
    }
    copy_pages(pool, layers, layer_stride, page_bytes, src, dst, pairs);
}

__global__ void __launch_bounds__(256) kv4_free_kernel(PageArgs a, const uint32_t* slot_ids, uint32_t n)
{
    const uint64_t cells = (uint64_t)n * a.max_pages;
    for (uint64_t x = blockIdx.x * 256ull + threadIdx.x; x < cells; x += gridDim.x * 256ull)
    {
        const uint32_t i = (uint32_t)(x / a.max_pages), col = (uint32_t)(x % a.max_pages);
        const uint32_t slot = slot_ids ? slot_ids[i] : i;
        if (slot >= a.slots)
        {
            if (col == 0) atomicOr(a.status, (int)FML_KV4_BAD_SLOT);
            continue;
        }
        // whoever takes the entry gives the page back, so a slot named twice
        // is freed once
        const int32_t p = atomicExch(&a.table[(uint64_t)slot * a.max_pages + col], -1);
        if (p >= 0 && (uint32_t)p < a.pages) atomicSub(&a.refs[p], 1);
        if (col == 0) a.lens[slot] = 0;
    }
}

// compact: workspace lists holes[pages / 2 + 1], movers[...], to[pages] (the
// new number of a page that moves).
__global__ void __launch_bounds__(PT) kv4_compact_kernel(PageArgs a, uint32_t* ws)
{
    const uint32_t most = a.pages / 2 + 1;
    uint32_t* holes = ws + WS_HEAD;
    uint32_t* movers = holes + most;
    uint32_t* to = movers + most;
    uint32_t live = 0;
    for (uint32_t p0 = 0; p0 < a.pages; p0 += 4 * PT)
    {
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const uint32_t p = p0 + 4 * threadIdx.x + i;
            mine += p < a.pages && a.refs[p] > 0;
        }
        live += mine;
    }
    uint32_t total;
    block_exclusive(live, &total);
    live = total;
    uint32_t nh = 0, nm = 0;
    for (uint32_t p0 = 0; p0 < a.pages; p0 += 4 * PT)
    {
        const uint32_t p = p0 + 4 * threadIdx.x;
        bool listed[4];
        uint32_t hole = 0, move = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            const bool in = p + i < a.pages, used = in && a.refs[p + i] > 0;
            const bool low = p + i < live;
            listed[i] = in && used != low;
            if (listed[i]) (low ? hole : move) += 1;
            if (in && !low && !used) to[p + i] = p + i;  // a free page stays where it is
        }
        uint32_t th, tm;
        uint32_t ah = nh + block_exclusive(hole, &th), am = nm + block_exclusive(move, &tm);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (listed[i])
            {
                if (p + i < live) holes[ah++] = p + i;
                else movers[am++] = p + i;
            }
        nh += th;
        nm += tm;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < nm; i += PT)
    {
        const uint32_t m = movers[i], h = holes[i];
        to[m] = h;
        a.refs[h] = a.refs[m];
        a.refs[m] = 0;
    }
    if (threadIdx.x == 0)
    {
        ws[0] = nm;
        ws[1] = live;
    }
}

__global__ void __launch_bounds__(256) kv4_compact_copy_kernel(PageArgs a, unsigned char* pool, uint32_t layers,
                                                               uint64_t layer_stride, uint64_t page_bytes,
                                                               const uint32_t* ws)
{
    const uint32_t pairs = ws[0], live = ws[1];
    const uint32_t most = a.pages / 2 + 1;
    const uint32_t* holes = ws + WS_HEAD;
    const uint32_t* movers = holes + most;
    const uint32_t* to = movers + most;
    if (pairs == 0) return;
    const uint64_t cells = (uint64_t)a.slots * a.max_pages;
    for (uint64_t x = blockIdx.x * 256ull + threadIdx.x; x < cells; x += gridDim.x * 256ull)
    {
        const int32_t p = a.table[x];
        // entries name used pages; one past `live` has moved
        if (p >= 0 && (uint32_t)p >= live && (uint32_t)p < a.pages) a.table[x] = (int32_t)to[p];
    }
    copy_pages(pool, layers, layer_stride, page_bytes, movers, holes, pairs);
}

int check_pages(const char* who, const void* refs, const void* table, uint32_t pages, uint32_t slots,
                uint32_t max_pages, uint32_t n, const void* workspace, size_t workspace_bytes)
{
    FML_REQUIRE(refs && table, "%s: null pointer", who);
    FML_REQUIRE(pages >= 1 && pages <= MAX_PAGES && slots >= 1 && n < (1u << 30), "%s: %u pages, %u slots, %u entries",
                who, pages, slots, n);
    FML_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= fml_kv4_pages_workspace_bytes(pages, n),
                "%s: the workspace needs %zu bytes, 16-byte aligned", who, fml_kv4_pages_workspace_bytes(pages, n));
    return FML_OK;
}

int check_pool(const char* who, const void* pool, uint32_t layers, uint64_t layer_stride, uint64_t page_bytes,
               uint32_t pages)
{
    FML_REQUIRE(pool && aligned16(pool), "%s: the pool must be 16-byte aligned", who);
    FML_REQUIRE(layers >= 1 && page_bytes >= 16 && page_bytes % 16 == 0 && page_bytes < (1ull << 40) &&
                    layer_stride % 16 == 0 && (layers == 1 || layer_stride >= page_bytes * pages),
                "%s: %u layers %llu bytes apart, pages of %llu bytes", who, layers, (unsigned long long)layer_stride,
                (unsigned long long)page_bytes);
    return FML_OK;
}

int reserve_entry(const char* who, int32_t* refs, int32_t* table, uint32_t* lens, uint32_t* kept,
                  const uint32_t* slot_ids, const uint32_t* counts, uint32_t n, uint32_t pages, uint32_t slots,
                  uint32_t max_pages, uint32_t page_size, int32_t* status, void* workspace, size_t workspace_bytes,
                  cudaStream_t st)
{
    if (n == 0) return FML_OK;
    FML_RC(check_pages(who, refs, table, pages, slots, max_pages, n, workspace, workspace_bytes));
    FML_REQUIRE(lens && counts && status, "%s: null pointer", who);
    FML_REQUIRE(kv4_page_shift(page_size) && (uint64_t)max_pages * page_size < (1ull << 31),
                "%s: %u pages of %u rows a sequence", who, max_pages, page_size);
    const PageArgs a{refs, table, lens, pages, slots, max_pages, kv4_page_shift(page_size), status};
    kv4_reserve_kernel<<<1, PT, 0, st>>>(a, slot_ids, counts, n, kept, static_cast<uint32_t*>(workspace));
    FML_LAUNCH_CHECK();
    return FML_OK;
}

constexpr uint32_t COPY_CTAS = 148 * 8;

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" {

size_t fml_kv4_block_bytes(uint32_t head_dim, uint32_t page_size)
{
    if (!(head_dim == 32 || head_dim == 64 || head_dim == 128) || !kv4_page_shift(page_size)) return 0;
    return (size_t)page_size * head_dim * 5 / 4;
}

int fml_kv4_append(void* pool, const int32_t* table, const uint32_t* lens, const uint32_t* slot_ids, const void* k,
                   const void* v, int type, const uint32_t* starts, uint32_t batch, uint32_t rows, uint32_t ldk,
                   uint32_t ldv, uint32_t pages, uint32_t slots, uint32_t max_pages, uint32_t page_size,
                   uint32_t kv_heads, uint32_t head_dim, fml_stream_t stream)
{
    return rows_entry<false>("fml_kv4_append", pool, table, lens, slot_ids, nullptr, const_cast<void*>(k),
                             const_cast<void*>(v), type, starts, batch, rows, ldk, ldv, pages, slots, max_pages,
                             page_size, kv_heads, head_dim, as_stream(stream));
}

int fml_kv4_append_keeping(void* pool, const int32_t* table, const uint32_t* lens, const uint32_t* slot_ids,
                           const uint32_t* kept, const void* k, const void* v, int type, const uint32_t* starts,
                           uint32_t batch, uint32_t rows, uint32_t ldk, uint32_t ldv, uint32_t pages, uint32_t slots,
                           uint32_t max_pages, uint32_t page_size, uint32_t kv_heads, uint32_t head_dim,
                           fml_stream_t stream)
{
    if (batch == 0 || rows == 0) return FML_OK;
    FML_REQUIRE(kept, "fml_kv4_append_keeping: null pointer");
    return rows_entry<false>("fml_kv4_append_keeping", pool, table, lens, slot_ids, kept, const_cast<void*>(k),
                             const_cast<void*>(v), type, starts, batch, rows, ldk, ldv, pages, slots, max_pages,
                             page_size, kv_heads, head_dim, as_stream(stream));
}

int fml_kv4_read(void* k, void* v, int type, const void* pool, const int32_t* table, const uint32_t* lens,
                 const uint32_t* slot_ids, const uint32_t* starts, uint32_t batch, uint32_t rows, uint32_t ldk,
                 uint32_t ldv, uint32_t pages, uint32_t slots, uint32_t max_pages, uint32_t page_size,
                 uint32_t kv_heads, uint32_t head_dim, fml_stream_t stream)
{
    return rows_entry<true>("fml_kv4_read", const_cast<void*>(pool), table, lens, slot_ids, nullptr, k, v, type, starts,
                            batch, rows, ldk, ldv, pages, slots, max_pages, page_size, kv_heads, head_dim,
                            as_stream(stream));
}

size_t fml_kv4_pages_workspace_bytes(uint32_t pages, uint32_t n)
{
    const uint64_t lists = 5ull * n + 1 + (n ? pages : 0);        // reserve, fork
    const uint64_t moves = 2ull * (pages / 2 + 1) + pages;        // compact
    return (size_t)(4 * (WS_HEAD + (n ? lists : moves)) + 15) / 16 * 16;
}

int fml_kv4_reserve(int32_t* refs, int32_t* table, uint32_t* lens, const uint32_t* slot_ids, const uint32_t* counts,
                    uint32_t n, uint32_t pages, uint32_t slots, uint32_t max_pages, uint32_t page_size,
                    int32_t* status, void* workspace, size_t workspace_bytes, fml_stream_t stream)
{
    return reserve_entry("fml_kv4_reserve", refs, table, lens, nullptr, slot_ids, counts, n, pages, slots, max_pages,
                         page_size, status, workspace, workspace_bytes, as_stream(stream));
}

int fml_kv4_reserve_keeping(int32_t* refs, int32_t* table, uint32_t* lens, uint32_t* kept, const uint32_t* slot_ids,
                            const uint32_t* counts, uint32_t n, uint32_t pages, uint32_t slots, uint32_t max_pages,
                            uint32_t page_size, int32_t* status, void* workspace, size_t workspace_bytes,
                            fml_stream_t stream)
{
    if (n == 0) return FML_OK;
    FML_REQUIRE(kept, "fml_kv4_reserve_keeping: null pointer");
    return reserve_entry("fml_kv4_reserve_keeping", refs, table, lens, kept, slot_ids, counts, n, pages, slots,
                         max_pages, page_size, status, workspace, workspace_bytes, as_stream(stream));
}

int fml_kv4_fork(void* pool, uint32_t layers, uint64_t layer_stride, uint64_t page_bytes, int32_t* refs,
                 int32_t* table, uint32_t* lens, const uint32_t* parents, const uint32_t* children, uint32_t n,
                 uint32_t pages, uint32_t slots, uint32_t max_pages, uint32_t page_size, int32_t* status,
                 void* workspace, size_t workspace_bytes, fml_stream_t stream)
{
    if (n == 0) return FML_OK;
    FML_RC(check_pages("fml_kv4_fork", refs, table, pages, slots, max_pages, n, workspace, workspace_bytes));
    FML_RC(check_pool("fml_kv4_fork", pool, layers, layer_stride, page_bytes, pages));
    FML_REQUIRE(lens && parents && children && status, "fml_kv4_fork: null pointer");
    FML_REQUIRE(kv4_page_shift(page_size) && (uint64_t)max_pages * page_size < (1ull << 31),
                "fml_kv4_fork: %u pages of %u rows a sequence", max_pages, page_size);
    const PageArgs a{refs, table, lens, pages, slots, max_pages, kv4_page_shift(page_size), status};
    cudaStream_t st = as_stream(stream);
    uint32_t* ws = static_cast<uint32_t*>(workspace);
    kv4_fork_kernel<<<1, PT, 0, st>>>(a, parents, children, n, ws);
    FML_LAUNCH_CHECK();
    kv4_fork_copy_kernel<<<COPY_CTAS, 256, 0, st>>>(a, static_cast<unsigned char*>(pool), layers, layer_stride,
                                                    page_bytes, parents, children, n, ws);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

int fml_kv4_free(int32_t* refs, int32_t* table, uint32_t* lens, const uint32_t* slot_ids, uint32_t n, uint32_t pages,
                 uint32_t slots, uint32_t max_pages, int32_t* status, fml_stream_t stream)
{
    if (n == 0) return FML_OK;
    FML_REQUIRE(refs && table && lens && status, "fml_kv4_free: null pointer");
    FML_REQUIRE(pages >= 1 && slots >= 1 && max_pages >= 1, "fml_kv4_free: %u pages, %u slots of %u", pages, slots,
                max_pages);
    const PageArgs a{refs, table, lens, pages, slots, max_pages, 0, status};
    kv4_free_kernel<<<grid_for((uint64_t)n * max_pages, 256), 256, 0, as_stream(stream)>>>(a, slot_ids, n);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

int fml_kv4_compact(void* pool, uint32_t layers, uint64_t layer_stride, uint64_t page_bytes, int32_t* refs,
                    int32_t* table, uint32_t pages, uint32_t slots, uint32_t max_pages, void* workspace,
                    size_t workspace_bytes, fml_stream_t stream)
{
    FML_RC(check_pages("fml_kv4_compact", refs, table, pages, slots, max_pages, 0, workspace, workspace_bytes));
    FML_RC(check_pool("fml_kv4_compact", pool, layers, layer_stride, page_bytes, pages));
    const PageArgs a{refs, table, nullptr, pages, slots, max_pages, 0, nullptr};
    cudaStream_t st = as_stream(stream);
    uint32_t* ws = static_cast<uint32_t*>(workspace);
    kv4_compact_kernel<<<1, PT, 0, st>>>(a, ws);
    FML_LAUNCH_CHECK();
    kv4_compact_copy_kernel<<<COPY_CTAS, 256, 0, st>>>(a, static_cast<unsigned char*>(pool), layers, layer_stride,
                                                       page_bytes, ws);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

}  // extern "C"
