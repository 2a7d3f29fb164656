// Causal attention over packed prompts with grouped heads, on the CUDA cores:
// any strides and alignment.
//
// CTA = 256 threads, 16 x 16, on a tile of 64 query rows of one key/value head
// (packed.cuh); it walks the key tiles of 64 that its last token sees with an
// online softmax.  Thread (ty, tx) owns rows ty + 16 i, keys tx + 16 j of the
// score tile and output columns tx + 16 c.  fp32 throughout.  It is for what the
// tensor-core kernels cannot take (bases or strides that are not multiples of 16
// bytes, FML_MATH_FP32, a 16-bit scale that is not positive): bound by the
// multiply-adds and the shared-memory reads that feed them, 512 causal tokens of
// 8 heads of 64 take 61 us on a B200, where the tensor cores take 26 (fp32) and
// 16 (16 bit); at one token it is 10 us against 7 and 9.
#include <type_traits>

#include "packed.cuh"

namespace fml {

namespace {

constexpr int PQ = 64, PK = 64;

template <int HD>
constexpr uint32_t simt_smem()
{
    return (uint32_t)((PQ + 2 * PK) * (HD + 4) + PQ * (PK + 4)) * 4u;
}

template <typename T, int HD>
__global__ void __launch_bounds__(256) packed_attention_kernel(T* __restrict__ out, const T* __restrict__ q,
                                                               const T* __restrict__ k, const T* __restrict__ v,
                                                               PackedArgs a)
{
    constexpr int HP = HD + 4, OC = HD / 16;
    extern __shared__ __align__(16) float sm[];
    float* Qs = sm;
    float* Ks = Qs + PQ * HP;
    float* Vs = Ks + PK * HP;
    float* Ps = Vs + PK * HP;
    __shared__ PackedTile found;
    if (threadIdx.x < 32)
    {
        const PackedTile t = packed_tile(a, packed_totals(a), blockIdx.x / (a.kv_heads * a.nchunk));
        if (threadIdx.x == 0) found = t;
    }
    __syncthreads();
    const PackedTile p = found;
    if (!p.live) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const uint32_t y = blockIdx.x % (a.kv_heads * a.nchunk), kvh = y / a.nchunk, hc = (y % a.nchunk) * a.gs;
    const uint32_t nh = min(a.gs, a.group - hc);  // heads of this tile
    const uint32_t nt = min(a.tpt, p.lq - p.t0);  // tokens
    // row r: token p.t0 + r / gs, head hc + r % gs
    for (int i = tid; i < PQ * HD; i += 256)
    {
        const uint32_t r = i / HD, c = i % HD, t = r / a.gs, h = r % a.gs;
        float x = 0.f;
        if (t < nt && h < nh)
            x = to_f32(q[(uint64_t)(p.q0 + p.t0 + t) * a.ldq + (kvh * a.group + hc + h) * HD + c]) * a.scale;
        Qs[r * HP + c] = x;
    }
    uint32_t seen[4];
    float m[4], l[4], o[4][OC];
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const uint32_t r = ty + 16 * i, t = r / a.gs;
        seen[i] = t < nt && r % a.gs < nh ? keys_seen(p, p.t0 + t) : 0u;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < OC; ++c) o[i][c] = 0.f;
    }
    const uint32_t nkeys = keys_seen(p, p.t0 + nt - 1);
    for (uint32_t k0 = 0; k0 < nkeys; k0 += PK)
    {
        __syncthreads();
        for (int i = tid; i < PK * HD; i += 256)
        {
            const uint32_t r = i / HD, c = i % HD;
            const bool in = k0 + r < nkeys;
            const uint64_t row = p.k0 + k0 + r;
            Ks[r * HP + c] = in ? to_f32(k[row * a.ldk + kvh * HD + c]) : 0.f;
            Vs[r * HP + c] = in ? to_f32(v[row * a.ldv + kvh * HD + c]) : 0.f;
        }
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 4
        for (int e = 0; e < HD; e += 4)
        {
            float4 qv[4], kv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + (ty + 16 * i) * HP + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) kv[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * HP + e);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                {
                    s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
                    s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
                    s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
                    s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                s[i][j] = k0 + tx + 16 * j < seen[i] ? s[i][j] : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL_MASK, mx, w));
            const float corr = m[i] == -INFINITY ? 0.f : expf(m[i] - mx);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j)
            {
                const float e = s[i][j] == -INFINITY ? 0.f : expf(s[i][j] - mx);
                Ps[(ty + 16 * i) * (PK + 4) + tx + 16 * j] = e;
                sum += e;
            }
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) sum += __shfl_xor_sync(FULL_MASK, sum, w);
            l[i] = l[i] * corr + sum;
            m[i] = mx;
#pragma unroll
            for (int c = 0; c < OC; ++c) o[i][c] *= corr;
        }
        __syncwarp();  // a row's probabilities are written and read by one half-warp
#pragma unroll 4
        for (int j = 0; j < PK; ++j)
        {
            float pv[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pv[i] = Ps[(ty + 16 * i) * (PK + 4) + j];
#pragma unroll
            for (int c = 0; c < OC; ++c)
            {
                const float x = Vs[j * HP + tx + 16 * c];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i][c] = fmaf(pv[i], x, o[i][c]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
    {
        const uint32_t r = ty + 16 * i, t = r / a.gs, h = r % a.gs;
        if (t >= nt || h >= nh) continue;
        T* dst = out + (uint64_t)(p.q0 + p.t0 + t) * a.ldo + (kvh * a.group + hc + h) * HD;
        const float inv = seen[i] ? 1.0f / l[i] : 0.f;
#pragma unroll
        for (int c = 0; c < OC; ++c) dst[tx + 16 * c] = from_f32<T>(seen[i] ? o[i][c] * inv : 0.f);
    }
}

template <typename T, int HD>
int launch_simt(void* out, const void* q, const void* k, const void* v, PackedArgs a, cudaStream_t st)
{
    auto kern = packed_attention_kernel<T, HD>;
    static uint64_t attr_devices = 0;
    FML_RC(smem_limit_once(reinterpret_cast<const void*>(kern), (int)simt_smem<HD>(), attr_devices));
    const uint64_t blocks = packed_items(&a, PQ, 1);
    FML_REQUIRE(blocks < (1ull << 31), "fml_attention_packed: %u rows, %u heads", a.q_rows, a.heads);
    kern<<<(unsigned)blocks, 256, simt_smem<HD>(), st>>>(
        static_cast<T*>(out), static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v), a);
    FML_LAUNCH_CHECK();
    return FML_OK;
}

}  // namespace
}  // namespace fml

using namespace fml;

extern "C" int fml_attention_packed(void* out, const void* q, const void* k, const void* v, int type,
                                    const uint32_t* q_starts, const uint32_t* k_starts, uint32_t batch,
                                    uint32_t q_rows, uint32_t k_rows, uint32_t heads, uint32_t kv_heads,
                                    uint32_t head_dim, uint32_t ldo, uint32_t ldq, uint32_t ldk, uint32_t ldv,
                                    float scale, int mode, fml_stream_t stream)
{
    if (batch == 0 || q_rows == 0) return FML_OK;
    FML_REQUIRE(out && q && q_starts && (k_rows == 0 || (k && v)), "fml_attention_packed: null pointer");
    FML_REQUIRE(type == FML_TYPE_FP32 || type == FML_TYPE_FP16 || type == FML_TYPE_BF16,
                "fml_attention_packed: unknown type %d", type);
    FML_REQUIRE(head_dim == 32 || head_dim == 64 || head_dim == 128,
                "fml_attention_packed: head_dim %u (need 32, 64 or 128)", head_dim);
    FML_REQUIRE(kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0,
                "fml_attention_packed: %u query heads over %u key/value heads", heads, kv_heads);
    FML_REQUIRE((uint64_t)heads * head_dim <= ldq && (uint64_t)heads * head_dim <= ldo &&
                    (uint64_t)kv_heads * head_dim <= ldk && (uint64_t)kv_heads * head_dim <= ldv,
                "fml_attention_packed: %u and %u heads of %u, strides %u, %u, %u, %u", heads, kv_heads, head_dim, ldo,
                ldq, ldk, ldv);
    FML_REQUIRE(mode == FML_MATH_FP32 || mode == FML_MATH_TF32X3 || mode == FML_MATH_TF32,
                "fml_attention_packed: unknown math mode %d", mode);
    FML_REQUIRE(q_rows < (1u << 31) && k_rows < (1u << 31) && batch < (1u << 30),
                "fml_attention_packed: %u and %u rows, batch %u", q_rows, k_rows, batch);
    PackedArgs a{};
    a.q_starts = q_starts;
    a.k_starts = k_starts ? k_starts : q_starts;
    a.batch = batch;
    a.q_rows = q_rows;
    a.k_rows = k_rows;
    a.heads = heads;
    a.kv_heads = kv_heads;
    a.group = heads / kv_heads;
    a.ldo = ldo;
    a.ldq = ldq;
    a.ldk = ldk;
    a.ldv = ldv;
    a.scale = scale;
    cudaStream_t st = as_stream(stream);
    if (type != FML_TYPE_FP32)
    {
        const int rc = launch_packed_attention_tc(out, q, k, v, type, head_dim, a, st);
        if (rc != FML_ERR_UNSUPPORTED) return rc;
    }
    else if (mode != FML_MATH_FP32)
    {
        const int rc = launch_packed_attention_tf32(static_cast<float*>(out), static_cast<const float*>(q),
                                                    static_cast<const float*>(k), static_cast<const float*>(v), head_dim, a,
                                                    mode == FML_MATH_TF32X3, st);
        if (rc != FML_ERR_UNSUPPORTED) return rc;
    }
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (head_dim == 32) return launch_simt<T, 32>(out, q, k, v, a, st);
        if (head_dim == 64) return launch_simt<T, 64>(out, q, k, v, a, st);
        return launch_simt<T, 128>(out, q, k, v, a, st);
    };
    if (type == FML_TYPE_FP32) return go(static_cast<float*>(nullptr));
    if (type == FML_TYPE_FP16) return go(static_cast<__half*>(nullptr));
    return go(static_cast<__nv_bfloat16*>(nullptr));
}
