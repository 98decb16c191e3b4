// SPDX-License-Identifier: Apache-2.0
// Attention of new tokens over the paged generation cache.
//
// Query j of a sequence stands at position p = starts + j and sees the cached positions max(0, p - window + 1) .. p:
// o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m), s_t = scale q.k_t, in one pass over the keys with the running maximum m.
// The latent form has one key row [latent | rotary] for all heads and the latent itself as value.
#include "paged_common.cuh"

namespace atb {
namespace paged {

struct AttnArgs {
    const void *q, *q2;  // q [B, S, Hq, D1]; q2 [B, S, Hq, D - D1] (latent form) or null
    int64_t q_b, q_s, q_h, q2_b, q2_s, q2_h;
    const void *k_pages, *v_pages;
    const float *k_scale, *v_scale;
    int64_t k_page, v_page, ks_page, vs_page;
    void* out;  // [B, S, Hq, Dv]
    const int *table, *starts, *counts;
    int64_t table_stride;
    int S, Hq, Hkv, D, D1, Dv, P, W, page, window;
    float scale;
};

template <typename T, bool E4M3>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&f)[8]) {
    if (E4M3) unpack_e4m3x8(*reinterpret_cast<const uint2*>((const uint8_t*)base + at), f);
    else Vec8<T>::unpack(*reinterpret_cast<const uint4*>((const T*)base + at), f);
}

// One CTA per (sequence, new token, query head); its warps take keys in turn and are joined at the end.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(128) attention_kernel(const AttnArgs a) {
    constexpr int kMax = 3;  // chunks of 8 elements a lane: D <= 768
    __shared__ float s_m[4], s_l[4];
    __shared__ float s_o[4][512];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.Hq;
    const int64_t bj = blockIdx.x / a.Hq;
    const int64_t b = bj / a.S;
    const int j = (int)(bj - b * a.S);
    const int kvh = h / (a.Hq / a.Hkv);
    const int count = a.counts ? min(a.counts[b], a.S) : a.S;
    const int64_t pos = (int64_t)a.starts[b] + j;
    int64_t end = min(min(pos + 1, (int64_t)a.starts[b] + count), (int64_t)a.W * a.page);
    if (j >= count) end = 0;
    const int64_t first = a.window > 0 ? max((int64_t)0, pos + 1 - a.window) : 0;
    float q[kMax][8] = {}, o[kMax][8] = {};
    for (int i = 0; i < kMax; ++i) {
        const int e = (lane + 32 * i) * 8;
        if (e < a.D1) Vec8<T>::unpack(*reinterpret_cast<const uint4*>((const T*)a.q + b * a.q_b + j * a.q_s + h * a.q_h + e), q[i]);
        else if (e < a.D) Vec8<T>::unpack(*reinterpret_cast<const uint4*>((const T*)a.q2 + b * a.q2_b + j * a.q2_s + h * a.q2_h + e - a.D1), q[i]);
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t t = first + warp; t < end; t += 4) {
        const int w = (int)t / a.page, off = (int)t - w * a.page;
        const int pid = a.table[b * a.table_stride + w];
        if (pid < 0 || pid >= a.P) continue;
        const int64_t row = (int64_t)kvh * a.page + off;
        float dot = 0.f;
        for (int i = 0; i < kMax; ++i) {
            const int e = (lane + 32 * i) * 8;
            if (e < a.D) {
                float k[8];
                load8<T, E4M3>(a.k_pages, pid * a.k_page + row * a.D + e, k);
                for (int x = 0; x < 8; ++x) dot += q[i][x] * k[x];
            }
        }
        dot = warp_sum(dot) * a.scale;
        if (E4M3) dot *= a.k_scale[pid * a.ks_page + row];
        const float mn = max_nan(m, dot);
        const float c = m == -INFINITY ? 0.f : __expf(m - mn);
        const float p = mn == -INFINITY ? 0.f : __expf(dot - mn);
        m = mn;
        l = l * c + p;
        const float pv = E4M3 ? p * a.v_scale[pid * a.vs_page + row] : p;
        for (int i = 0; i < kMax; ++i) {
            const int e = (lane + 32 * i) * 8;
            if (e < a.Dv) {
                float v[8];
                load8<T, E4M3>(a.v_pages, pid * a.v_page + row * a.D + e, v);
                for (int x = 0; x < 8; ++x) o[i][x] = o[i][x] * c + pv * v[x];
            }
        }
    }
    if (lane == 0) {
        s_m[warp] = m;
        s_l[warp] = l;
    }
    for (int i = 0; i < kMax; ++i) {
        const int e = (lane + 32 * i) * 8;
        if (e < a.Dv)
            for (int x = 0; x < 8; ++x) s_o[warp][e + x] = o[i][x];
    }
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < 4; ++w) top = max_nan(top, s_m[w]);
    float total = 0.f, f[4];
    for (int w = 0; w < 4; ++w) {
        f[w] = s_m[w] == -INFINITY ? 0.f : __expf(s_m[w] - top);
        total += f[w] * s_l[w];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    for (int e = threadIdx.x * 8; e < a.Dv; e += 128 * 8) {
        float r[8];
        for (int x = 0; x < 8; ++x) {
            r[x] = 0.f;
            for (int w = 0; w < 4; ++w) r[x] += f[w] == 0.f ? 0.f : f[w] * s_o[w][e + x];
            r[x] *= inv;
        }
        *reinterpret_cast<uint4*>((T*)a.out + (bj * a.Hq + h) * a.Dv + e) = Vec8<T>::pack(r);
    }
}

static void launch_attention(const at::Tensor& q, bool f8, const AttnArgs& a, int64_t B) {
    cudaStream_t st = current_stream();
    const dim3 grid((unsigned)(B * a.S * a.Hq));
    if (q.scalar_type() == at::kBFloat16) {
        if (f8) attention_kernel<bf16, true><<<grid, 128, 0, st>>>(a);
        else attention_kernel<bf16, false><<<grid, 128, 0, st>>>(a);
    } else {
        if (f8) attention_kernel<__half, true><<<grid, 128, 0, st>>>(a);
        else attention_kernel<__half, false><<<grid, 128, 0, st>>>(a);
    }
    ATB_LAUNCH_CHECK();
}

static bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

}  // namespace paged

using namespace paged;

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages, const at::Tensor& table,
                           const at::Tensor& starts, const c10::optional<at::Tensor>& counts,
                           const c10::optional<at::Tensor>& k_scale, const c10::optional<at::Tensor>& v_scale, double scale,
                           int64_t window) {
    const char* op = "paged_attention";
    ATB_ARG(q.dim() == 4, op, ": q must be [batch, new tokens, heads, dim]");
    const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2), D = q.size(3);
    ATB_ARG(half_type(q), op, ": q must be bf16 or fp16");
    ATB_ARG(D % 16 == 0 && D <= 256 && D > 0, op, ": dim must be a multiple of 16 up to 256");
    check_pages(op, k_pages, k_scale, q);
    check_pages(op, v_pages, v_scale, q);
    ATB_ARG(k_pages.sizes() == v_pages.sizes() && k_pages.scalar_type() == v_pages.scalar_type(), op, ": k_pages and v_pages differ");
    const int64_t Hkv = k_pages.size(1);
    ATB_ARG(Hkv > 0 && Hq % Hkv == 0, op, ": the query heads must be a multiple of the cache's heads");
    ATB_ARG(k_pages.size(3) == D, op, ": the cache has another dim than q");
    ATB_ARG(is_e4m3(k_pages) || k_pages.scalar_type() == q.scalar_type(), op, ": the cache must have the query's type or be e4m3");
    ATB_ARG(window >= 0 && window < (int64_t(1) << 31), op, ": window must be positive");
    check_table(op, table, starts, counts, k_pages, B);
    ATB_ARG(B * S * Hq < (int64_t(1) << 31), op, ": too many query rows");
    const c10::cuda::CUDAGuard guard(q.device());
    at::Tensor out = at::empty({B, S, Hq, D}, q.options());
    if (out.numel() == 0) return out;
    const at::Tensor qc = rows16(q);
    AttnArgs a;
    a.q = qc.data_ptr(); a.q2 = nullptr;
    a.q_b = qc.stride(0); a.q_s = qc.stride(1); a.q_h = qc.stride(2); a.q2_b = a.q2_s = a.q2_h = 0;
    a.k_pages = k_pages.data_ptr(); a.v_pages = v_pages.data_ptr();
    a.k_scale = ptr<float>(k_scale); a.v_scale = ptr<float>(v_scale);
    a.k_page = k_pages.stride(0); a.v_page = v_pages.stride(0);
    a.ks_page = k_scale.has_value() ? k_scale->stride(0) : 0; a.vs_page = v_scale.has_value() ? v_scale->stride(0) : 0;
    a.out = out.data_ptr();
    a.table = table.data_ptr<int>(); a.starts = starts.data_ptr<int>(); a.counts = ptr<int>(counts);
    a.table_stride = table.stride(0);
    a.S = (int)S; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = a.D1 = a.Dv = (int)D; a.P = (int)k_pages.size(0); a.W = (int)table.size(1);
    a.page = (int)k_pages.size(2); a.window = (int)window; a.scale = (float)scale;
    launch_attention(q, is_e4m3(k_pages), a, B);
    return out;
}

at::Tensor paged_latent_attention(const at::Tensor& q, const at::Tensor& q_pe, const at::Tensor& pages, const at::Tensor& table,
                                  const at::Tensor& starts, const c10::optional<at::Tensor>& counts,
                                  const c10::optional<at::Tensor>& page_scale, double scale) {
    const char* op = "paged_latent_attention";
    ATB_ARG(q.dim() == 4 && q_pe.dim() == 4, op, ": q_latent and q_pe must be [batch, new tokens, heads, width]");
    const int64_t B = q.size(0), S = q.size(1), H = q.size(2), R = q.size(3), rope = q_pe.size(3);
    ATB_ARG(q_pe.size(0) == B && q_pe.size(1) == S && q_pe.size(2) == H, op, ": q_latent and q_pe differ in shape");
    ATB_ARG(half_type(q) && q_pe.scalar_type() == q.scalar_type(), op, ": q_latent and q_pe must be bf16 or fp16, both of one type");
    ATB_ARG(R % 16 == 0 && R > 0 && R <= 512 && rope % 16 == 0 && rope > 0 && rope <= 64, op,
            ": the latent must be a multiple of 16 up to 512, the rotary part one up to 64");
    ATB_ARG(q_pe.device() == q.device(), op, ": all tensors must be on one device");
    check_pages(op, pages, page_scale, q);
    ATB_ARG(pages.size(1) == 1 && pages.size(3) == R + rope, op, ": a latent cache is [pages, 1, page, latent + rotary]");
    ATB_ARG(is_e4m3(pages) || pages.scalar_type() == q.scalar_type(), op, ": the cache must have the query's type or be e4m3");
    check_table(op, table, starts, counts, pages, B);
    ATB_ARG(B * S * H < (int64_t(1) << 31), op, ": too many query rows");
    const c10::cuda::CUDAGuard guard(q.device());
    at::Tensor out = at::empty({B, S, H, R}, q.options());
    if (out.numel() == 0) return out;
    const at::Tensor qc = rows16(q), pc = rows16(q_pe);
    AttnArgs a;
    a.q = qc.data_ptr(); a.q2 = pc.data_ptr();
    a.q_b = qc.stride(0); a.q_s = qc.stride(1); a.q_h = qc.stride(2);
    a.q2_b = pc.stride(0); a.q2_s = pc.stride(1); a.q2_h = pc.stride(2);
    a.k_pages = a.v_pages = pages.data_ptr();
    a.k_scale = a.v_scale = ptr<float>(page_scale);
    a.k_page = a.v_page = pages.stride(0);
    a.ks_page = a.vs_page = page_scale.has_value() ? page_scale->stride(0) : 0;
    a.out = out.data_ptr();
    a.table = table.data_ptr<int>(); a.starts = starts.data_ptr<int>(); a.counts = ptr<int>(counts);
    a.table_stride = table.stride(0);
    a.S = (int)S; a.Hq = (int)H; a.Hkv = 1; a.D = (int)(R + rope); a.D1 = a.Dv = (int)R; a.P = (int)pages.size(0);
    a.W = (int)table.size(1); a.page = (int)pages.size(2); a.window = 0; a.scale = (float)scale;
    launch_attention(q, is_e4m3(pages), a, B);
    return out;
}

}  // namespace atb
