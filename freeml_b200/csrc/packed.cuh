// Packed prompts: which rows a CTA's tile of the packed attention holds.
//
// A tile is `rows` query rows of one key/value head: tokens in order, and for
// each the query heads of the group (row = token * gs + head), so that a group
// shares its key and value tiles.
#pragma once

#include "kv4.cuh"

namespace fml {

struct PackedArgs
{
    const uint32_t* q_starts;
    const uint32_t* k_starts;
    uint32_t batch, q_rows, k_rows;
    uint32_t heads, kv_heads;
    uint32_t group;         // query heads of a key/value head
    uint32_t gs, nchunk;    // query heads of a tile, tiles a token's group needs
    uint32_t tpt;           // tokens of a tile
    uint32_t step;          // tokens of a work item: one tile or two
    uint32_t mul, shift;    // x / step = x * mul >> shift for x < 2^31
    uint32_t ldo, ldq, ldk, ldv;
    float scale;
};

struct PackedTile
{
    uint32_t q0, k0;   // the sequence's first query and key row
    uint32_t lq, lk;   // its rows
    uint32_t t0;       // the tile's first token
    uint32_t live;     // 0: no tile of this number
};

__device__ __forceinline__ uint32_t clamped_rows(const uint32_t* starts, uint32_t b, uint32_t rows, uint32_t* first)
{
    const uint32_t s = min(starts[b], rows), e = min(starts[b + 1], rows);
    *first = s;
    return e > s ? e - s : 0u;
}

// Sequence b's rows; its work items weigh shift .. shift + n - 1: item j of a
// sequence weighs j and the keys before its first query, in items' tokens.
__device__ __forceinline__ void packed_sequence(const PackedArgs& a, uint32_t b, PackedTile* t, uint32_t* n,
                                                uint32_t* shift)
{
    *n = *shift = 0;
    if (b >= a.batch) return;
    auto steps = [&](uint32_t x) { return (uint32_t)((uint64_t)x * a.mul >> a.shift); };
    t->lq = clamped_rows(a.q_starts, b, a.q_rows, &t->q0);
    *n = steps(t->lq + a.step - 1);
    t->lk = t->lq;
    t->k0 = t->q0;
    if (a.k_starts == a.q_starts && a.k_rows == a.q_rows) return;
    t->lk = clamped_rows(a.k_starts, b, a.k_rows, &t->k0);
    if (t->lk > t->lq) *shift = steps(t->lk - t->lq);
}

// The number of items, and what they all weigh less than; by a whole warp.
struct PackedTotals
{
    uint32_t items, top;
};

__device__ inline PackedTotals packed_totals(const PackedArgs& a)
{
    PackedTile t;
    uint32_t n, shift, top = 0, total = 0;
#pragma unroll 4
    for (uint32_t b = threadIdx.x & 31u; b < a.batch; b += 32)
    {
        packed_sequence(a, b, &t, &n, &shift);
        total += n;
        if (n) top = max(top, n + shift);
    }
    return {__reduce_add_sync(FULL_MASK, total), __reduce_max_sync(FULL_MASK, top)};
}

// Item number `idx`'s rows: the heaviest items come first (among equals, the
// sequences in order), so that no long one is left for the end (sequence after
// sequence instead, each from its longest item on: 32 ragged fp32 prompts of up to
// 511 48 us, so 37, 64 of them 67 us, so 55; 12 grouped bf16 prompts of up to 4096
// 330 us, so 288; but 256 bf16 ones of up to 64 tokens, where the order is nothing
// and the search is what a short item waits for, 59, so 64; every item looks at all
// sequences, so that 4096 prompts of 16 tokens take 2.3 ms in bf16, where 1024 take
// 0.24: more are better split into calls).  A bisection finds the weight from the sequences'
// lengths.  Called by a whole warp.
__device__ inline PackedTile packed_tile(const PackedArgs& a, const PackedTotals& all, uint32_t idx)
{
    if (idx >= all.items) return PackedTile{};
    const uint32_t lane = threadIdx.x & 31u;
    PackedTile t{};
    uint32_t n, shift, lo = 0, hi = all.top, before = 0;
    // more than `idx` items weigh lo or more, `before` <= idx weigh hi or more
    while (hi - lo > 1)
    {
        const uint32_t mid = lo + (hi - lo) / 2;
        uint32_t sum = 0;
#pragma unroll 4
        for (uint32_t b = lane; b < a.batch; b += 32)
        {
            packed_sequence(a, b, &t, &n, &shift);
            if (n + shift > mid) sum += min(n, n + shift - mid);
        }
        sum = __reduce_add_sync(FULL_MASK, sum);
        if (sum > idx) lo = mid;
        else hi = mid, before = sum;
    }
    uint32_t left = idx - before;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 32)
    {
        packed_sequence(a, b0 + lane, &t, &n, &shift);
        const bool has = lo >= shift && lo - shift < n;
        const uint32_t with = __ballot_sync(FULL_MASK, has);
        if (left < (uint32_t)__popc(with))
        {
            const uint32_t ranked = __popc(with & ((1u << lane) - 1u));
            const int src = __ffs(__ballot_sync(FULL_MASK, has && ranked == left)) - 1;
            t.q0 = __shfl_sync(FULL_MASK, t.q0, src);
            t.k0 = __shfl_sync(FULL_MASK, t.k0, src);
            t.lq = __shfl_sync(FULL_MASK, t.lq, src);
            t.lk = __shfl_sync(FULL_MASK, t.lk, src);
            t.t0 = (lo - __shfl_sync(FULL_MASK, shift, src)) * a.step;
            t.live = 1;
            return t;
        }
        left -= __popc(with);
    }
    return PackedTile{};
}

// Keys that the tile's token t sees.
__device__ __forceinline__ uint32_t keys_seen(const PackedTile& p, uint32_t t)
{
    const int64_t n = (int64_t)t + 1 + p.lk - p.lq;
    return n <= 0 ? 0u : (uint32_t)(n < (int64_t)p.lk ? n : p.lk);
}

// Sets the split into tiles of `rows` rows, `tiles` of them to a work item, and
// gives the number of items at most: every sequence's last one may be part full.
inline uint64_t packed_items(PackedArgs* a, uint32_t rows, uint32_t tiles)
{
    a->gs = a->group < rows ? a->group : rows;
    a->nchunk = (a->group + a->gs - 1) / a->gs;
    a->tpt = rows / a->gs;
    a->step = tiles * a->tpt;
    a->shift = 31;  // mul = 2^shift / step rounded up: exact while its excess times x stays below 2^shift
    while ((1u << (a->shift - 31)) < a->step) ++a->shift;
    a->mul = (uint32_t)(((1ull << a->shift) + a->step - 1) / a->step);
    return ((uint64_t)a->q_rows / a->step + a->batch) * a->kv_heads * a->nchunk;
}

int launch_packed_attention_tc(void* out, const void* q, const void* k, const void* v, int type, uint32_t head_dim,
                               const PackedArgs& a, cudaStream_t st);
int launch_packed_attention_tf32(float* out, const float* q, const float* k, const float* v, uint32_t hd,
                                 const PackedArgs& p, bool split3, cudaStream_t st);

}  // namespace fml
