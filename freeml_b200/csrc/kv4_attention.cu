// Attention of one query row per sequence over the 4-bit paged cache.
//
// One CTA per (key/value head, sequence, up to 8 of its query heads); its
// warps take the keys in turn.  A lane has one column of each group of 32, so
// that it holds one code and one pair a group; scores are warp sums, and each
// warp keeps its own running maximum, sum and output.
#include <type_traits>

#include "kv4.cuh"

namespace fml {
namespace {

constexpr int GQ = 8;  // query heads of a CTA
constexpr int NW = 8;  // warps

template <typename T>
struct Kv4AttnArgs
{
    T* out;
    const T* q;
    uint32_t ldo, ldq;
    const unsigned char* pool;
    uint32_t group;  // query heads of a key/value head
    float scale;
    Kv4View c;
};

template <typename T, int HD>
__global__ void __launch_bounds__(32 * NW) kv4_attention_kernel(Kv4AttnArgs<T> a)
{
    using B = Kv4Block<HD>;
    constexpr int NG = B::NG;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t kvh = blockIdx.x, b = blockIdx.y, g0 = blockIdx.z * GQ;
    const uint32_t slot = kv4_slot(a.c, b), len = kv4_len(a.c, slot);
    const uint32_t nq = min((uint32_t)GQ, a.group - g0);
    const uint32_t page_size = 1u << a.c.page_shift;
    const uint32_t h0 = kvh * a.group + g0;

    float q[GQ][NG], o[GQ][NG], m[GQ], l[GQ];
#pragma unroll
    for (int i = 0; i < GQ; ++i)
    {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
        {
            o[i][g] = 0.f;
            q[i][g] = (uint32_t)i < nq ? to_f32(a.q[(uint64_t)b * a.ldq + (h0 + i) * HD + 32 * g + lane]) * a.scale : 0.f;
        }
    }
    for (uint32_t t = warp; t < len; t += NW)
    {
        const int32_t page = a.c.table[(uint64_t)slot * a.c.max_pages + (t >> a.c.page_shift)];
        if (page < 0 || (uint32_t)page >= a.c.pages) continue;
        const unsigned char* blk = a.pool + ((uint64_t)page * a.c.kv_heads + kvh) * B::bytes(page_size);
        const uint32_t row = t & (page_size - 1u);
        float k[NG], v[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g)
        {
            const uint32_t kw = reinterpret_cast<const uint32_t*>(blk + row * B::ROW)[(lane >> 3) * NG + g];
            const uint32_t vu =
                reinterpret_cast<const uint16_t*>(blk + B::v(page_size) + row * B::ROW)[(lane >> 2) * NG + g];
            const float2 km =
                __half22float2(reinterpret_cast<const __half2*>(blk + B::kmeta(page_size) + row * B::META)[g]);
            const float2 vm =
                __half22float2(reinterpret_cast<const __half2*>(blk + B::vmeta(page_size) + row * B::META)[g]);
            k[g] = fmaf((float)((kw >> (4 * (lane & 7u))) & 15u), km.x, km.y);
            v[g] = fmaf((float)((vu >> (4 * (lane & 3u))) & 15u), vm.x, vm.y);
        }
#pragma unroll
        for (int i = 0; i < GQ; ++i)
        {
            float s = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) s = fmaf(q[i][g], k[g], s);
            s = warp_sum(s);
            const float mn = fmaxf(m[i], s), corr = m[i] == -INFINITY ? 0.f : expf(m[i] - mn), p = expf(s - mn);
            l[i] = l[i] * corr + p;
#pragma unroll
            for (int g = 0; g < NG; ++g) o[i][g] = o[i][g] * corr + p * v[g];
            m[i] = mn;
        }
    }
    __shared__ float ms[NW][GQ], ls[NW][GQ], os[NW][HD];
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < GQ; ++i)
        {
            ms[warp][i] = m[i];
            ls[warp][i] = l[i];
        }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < GQ; ++i)
    {
        float top = -INFINITY, total = 0.f;
        for (int w = 0; w < NW; ++w) top = fmaxf(top, ms[w][i]);
        for (int w = 0; w < NW; ++w) total += ms[w][i] == -INFINITY ? 0.f : ls[w][i] * expf(ms[w][i] - top);
        const float f = m[i] == -INFINITY ? 0.f : expf(m[i] - top);
#pragma unroll
        for (int g = 0; g < NG; ++g) os[warp][32 * g + lane] = o[i][g] * f;
        __syncthreads();
        if ((uint32_t)i < nq)
            for (uint32_t d = threadIdx.x; d < HD; d += 32 * NW)
            {
                float s = 0.f;
                for (int w = 0; w < NW; ++w) s += os[w][d];
                a.out[(uint64_t)b * a.ldo + (h0 + i) * HD + d] = from_f32<T>(total == 0.f ? 0.f : s / total);
            }
        __syncthreads();
    }
}

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" {

size_t fml_attention_kv4_workspace_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }

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
    FML_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128, "fml_attention_kv4: head_dim %u", head_dim);
    FML_REQUIRE(kv4_page_shift(page_size) && (uint64_t)max_pages * page_size < (1ull << 31),
                "fml_attention_kv4: %u pages of %u rows a sequence", max_pages, page_size);
    FML_REQUIRE(pages >= 1 && pages < (1u << 31) && slots >= 1, "fml_attention_kv4: %u pages, %u slots", pages, slots);
    FML_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0,
                "fml_attention_kv4: %u query heads over %u key/value heads", heads, kv_heads);
    FML_REQUIRE((uint64_t)heads * head_dim <= ldq && (uint64_t)heads * head_dim <= ldo,
                "fml_attention_kv4: rows of %u heads of %u, strides %u and %u", heads, head_dim, ldq, ldo);
    const Kv4View c{table, lens, slot_ids, pages, slots, max_pages, kv4_page_shift(page_size), kv_heads};
    const uint32_t group = heads / kv_heads;
    const dim3 grid(kv_heads, batch, (group + GQ - 1) / GQ);
    FML_REQUIRE(batch <= 65535u && grid.z <= 65535u, "fml_attention_kv4: batch %u, group %u", batch, group);
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const Kv4AttnArgs<T> a{static_cast<T*>(out), static_cast<const T*>(q), ldo, ldq,
                               static_cast<const unsigned char*>(pool), group, scale, c};
        if (head_dim == 32) kv4_attention_kernel<T, 32><<<grid, 32 * NW, 0, as_stream(stream)>>>(a);
        else if (head_dim == 64) kv4_attention_kernel<T, 64><<<grid, 32 * NW, 0, as_stream(stream)>>>(a);
        else kv4_attention_kernel<T, 128><<<grid, 32 * NW, 0, as_stream(stream)>>>(a);
        FML_LAUNCH_CHECK();
        return (int)FML_OK;
    };
    if (type == FML_TYPE_FP32) return go(static_cast<float*>(nullptr));
    if (type == FML_TYPE_FP16) return go(static_cast<__half*>(nullptr));
    return go(static_cast<__nv_bfloat16*>(nullptr));
}

}  // extern "C"
