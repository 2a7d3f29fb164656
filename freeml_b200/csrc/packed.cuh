// Packed prompts: which rows a CTA's tile of the packed attention holds.
//
// A tile is `rows` query rows of one key/value head: tokens in order, and for
// each the query heads of the group (row = token * gs + head), so that a group
// shares its key and value tiles.  Tiles are numbered over the sequences by a
// block scan of their tile counts; the number is turned round, so that within
// a sequence the tiles with the most keys come first.
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

// The tile of number `idx` (of all tiles, the last first); called by every
// thread of a CTA of NT threads.
template <int NT>
__device__ PackedTile packed_tile(const PackedArgs& a, uint32_t idx)
{
    __shared__ uint32_t warp_s[NT / 32];
    __shared__ PackedTile tile_s;
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
    if (tid == 0) tile_s.live = 0;
    const uint32_t per = (a.batch + NT - 1) / NT, b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    uint32_t mine = 0, first;
    for (uint32_t b = b0; b < b1; ++b) mine += (clamped_rows(a.q_starts, b, a.q_rows, &first) + a.tpt - 1) / a.tpt;
    uint32_t x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
        if (lane >= (uint32_t)o) x += y;
    }
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    uint32_t before = x - mine, total = 0;
    for (uint32_t w = 0; w < NT / 32; ++w)
    {
        if (w < warp) before += warp_s[w];
        total += warp_s[w];
    }
    if (idx < total)
    {
        uint32_t left = total - 1 - idx;  // counted from the front
        if (left >= before && left < before + mine)
        {
            left -= before;
            for (uint32_t b = b0; b < b1; ++b)
            {
                PackedTile t;
                t.lq = clamped_rows(a.q_starts, b, a.q_rows, &t.q0);
                const uint32_t n = (t.lq + a.tpt - 1) / a.tpt;
                if (left < n)
                {
                    t.lk = clamped_rows(a.k_starts, b, a.k_rows, &t.k0);
                    t.t0 = left * a.tpt;
                    t.live = 1;
                    tile_s = t;
                    break;
                }
                left -= n;
            }
        }
    }
    __syncthreads();
    return tile_s;
}

// The tile of number `idx` of all tiles, sequence after sequence, each from its
// last tile to its first; called by a whole warp.
__device__ inline PackedTile packed_tile_warp(const PackedArgs& a, uint32_t idx)
{
    const uint32_t lane = threadIdx.x & 31u;
    PackedTile t{};
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 32)
    {
        const uint32_t b = b0 + lane;
        uint32_t q0 = 0, n = 0, lq = 0;
        if (b < a.batch)
        {
            lq = clamped_rows(a.q_starts, b, a.q_rows, &q0);
            n = (lq + a.tpt - 1) / a.tpt;
        }
        uint32_t x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const uint32_t y = __shfl_up_sync(FULL_MASK, x, o);
            if (lane >= (uint32_t)o) x += y;
        }
        const uint32_t found = __ballot_sync(FULL_MASK, idx < x);
        if (found)
        {
            const int src = __ffs(found) - 1;
            t.q0 = __shfl_sync(FULL_MASK, q0, src);
            t.lq = __shfl_sync(FULL_MASK, lq, src);
            t.t0 = (__shfl_sync(FULL_MASK, x, src) - 1 - idx) * a.tpt;
            t.lk = clamped_rows(a.k_starts, b0 + (uint32_t)src, a.k_rows, &t.k0);
            t.live = 1;
            return t;
        }
        idx -= __shfl_sync(FULL_MASK, x, 31);
    }
    return t;
}

// Keys that the tile's token t sees.
__device__ __forceinline__ uint32_t keys_seen(const PackedTile& p, uint32_t t)
{
    const int64_t n = (int64_t)t + 1 + p.lk - p.lq;
    return n <= 0 ? 0u : (uint32_t)(n < (int64_t)p.lk ? n : p.lk);
}

// Tiles at most: every sequence's last one may be part full.
inline uint64_t packed_tiles_bound(const PackedArgs& a) { return (uint64_t)a.q_rows / a.tpt + a.batch; }

int launch_packed_attention_tc(void* out, const void* q, const void* k, const void* v, int type, uint32_t head_dim,
                               const PackedArgs& a, cudaStream_t st);
int launch_packed_attention_tf32(float* out, const float* q, const float* k, const float* v, uint32_t hd,
                                 const PackedArgs& p, bool split3, cudaStream_t st);

}  // namespace fml
