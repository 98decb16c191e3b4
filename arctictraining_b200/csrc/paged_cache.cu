// SPDX-License-Identifier: Apache-2.0
// Writing and reading the paged generation cache: rotation of queries and keys fused with the write of keys and values
// (plain or e4m3), the same for latent rows with their RMS norm, and the read-back into dense tensors.
// All of it is bound by memory traffic: every input is read once and every output written once, in 16-byte accesses.
#include "paged_common.cuh"

namespace atb {
namespace paged {

// Where the new token (b, j) goes: page id and offset, or false when it is not written.
__device__ __forceinline__ bool find_slot(const int* __restrict__ table, int64_t table_stride, int W, int P, int page, int start,
                                          int j, int count, int64_t b, int& pid, int& off) {
    if (j >= count || start < 0) return false;
    const int64_t pos = (int64_t)start + j;
    if (pos >= (int64_t)W * page) return false;
    const int w = (int)pos / page;
    pid = table[b * table_stride + w];
    off = (int)pos - w * page;
    return pid >= 0 && pid < P;
}

struct AppendArgs {
    const void *q, *k, *v;
    int64_t q_b, q_s, q_h, k_b, k_s, k_h, v_b, v_s, v_h;  // strides in elements
    const float *cos, *sin;                                // [B, S, D / 2]
    void* q_out;                                           // [B, S, Hq, D]
    void *k_pages, *v_pages;
    float *k_scale, *v_scale;
    int64_t k_page, v_page, ks_page, vs_page;  // strides of one page in elements
    const int *table, *starts, *counts;
    int64_t table_stride;
    int S, Hq, Hkv, D, P, W, page;
};

// One CTA per new token.  A group of `LPR` lanes (a power of two >= D / 16) owns one head's row at a time; lane i of it holds
// elements [8 i, 8 i + 8) of both halves, so a rotation pair (i, i + D / 2) and its cos / sin stay in one thread.  The cos /
// sin of a lane are loaded once and serve all heads of the token.
template <typename T, bool E4M3, int LPR>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    const int64_t tok = blockIdx.x;
    const int64_t b = tok / a.S;
    const int j = (int)(tok - b * a.S);
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
    constexpr int kGroups = 256 / LPR;
    const int half = a.D / 2;
    const bool active = lane * 8 < half;
    float c[8], s[8];
    if (active) {
        const float4* pc = reinterpret_cast<const float4*>(a.cos + tok * half + lane * 8);
        const float4* ps = reinterpret_cast<const float4*>(a.sin + tok * half + lane * 8);
        const float4 c0 = pc[0], c1 = pc[1], s0 = ps[0], s1 = ps[1];
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
        s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
    }
    int pid = 0, off = 0;
    const bool keep = find_slot(a.table, a.table_stride, a.W, a.P, a.page, a.starts[b], j,
                                a.counts ? a.counts[b] : a.S, b, pid, off);
    const int rows = keep ? a.Hq + 2 * a.Hkv : a.Hq;
    // every lane of a warp takes the same number of rounds, so the shuffles below are complete
    for (int r0 = 0; r0 < rows; r0 += kGroups) {
        const int r = r0 + group;
        const bool mine = r < rows && active;
        const int kind = r < a.Hq ? 0 : (r < a.Hq + a.Hkv ? 1 : 2);
        float x[8] = {}, y[8] = {};
        if (mine) {
            const T* src;
            if (kind == 0) src = (const T*)a.q + b * a.q_b + j * a.q_s + r * a.q_h;
            else if (kind == 1) src = (const T*)a.k + b * a.k_b + j * a.k_s + (r - a.Hq) * a.k_h;
            else src = (const T*)a.v + b * a.v_b + j * a.v_s + (r - a.Hq - a.Hkv) * a.v_h;
            Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + lane * 8), x);
            Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + half + lane * 8), y);
            if (kind != 2) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float u = x[i], w = y[i];
                    x[i] = u * c[i] - w * s[i];
                    y[i] = w * c[i] + u * s[i];
                }
            }
        }
        float inv = 1.f, scale = 1.f;
        if (E4M3) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max_nan(m, max_nan(fabsf(x[i]), fabsf(y[i])));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            scale = e4m3_scale(m);
            inv = __fdiv_rn(1.f, scale);
        }
        if (!mine) continue;
        if (kind == 0) {
            T* dst = (T*)a.q_out + (tok * a.Hq + r) * a.D;
            *reinterpret_cast<uint4*>(dst + lane * 8) = Vec8<T>::pack(x);
            *reinterpret_cast<uint4*>(dst + half + lane * 8) = Vec8<T>::pack(y);
            continue;
        }
        const int h = kind == 1 ? r - a.Hq : r - a.Hq - a.Hkv;
        const int64_t row = (int64_t)h * a.page + off;
        if (E4M3) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] *= inv;
                y[i] *= inv;
            }
            uint8_t* dst = (uint8_t*)(kind == 1 ? a.k_pages : a.v_pages) + pid * (kind == 1 ? a.k_page : a.v_page) + row * a.D;
            *reinterpret_cast<uint2*>(dst + lane * 8) = pack_e4m3x8(x);
            *reinterpret_cast<uint2*>(dst + half + lane * 8) = pack_e4m3x8(y);
            if (lane == 0) (kind == 1 ? a.k_scale : a.v_scale)[pid * (kind == 1 ? a.ks_page : a.vs_page) + row] = scale;
        } else {
            T* dst = (T*)(kind == 1 ? a.k_pages : a.v_pages) + pid * (kind == 1 ? a.k_page : a.v_page) + row * a.D;
            *reinterpret_cast<uint4*>(dst + lane * 8) = Vec8<T>::pack(x);
            *reinterpret_cast<uint4*>(dst + half + lane * 8) = Vec8<T>::pack(y);
        }
    }
}

struct LatentAppendArgs {
    const void *q, *a, *w;  // q [B, S, H, rope] strided, a [B, S, R + rope] strided, w [R]
    int64_t q_b, q_s, q_h, a_b, a_s;
    const float *cos, *sin;  // [B, S, rope / 2]
    void* q_out;             // [B, S, H, rope]
    void* pages;
    float* scale;
    int64_t page_stride, scale_stride;
    const int *table, *starts, *counts;
    int64_t table_stride;
    float eps;
    int S, H, R, rope, P, W, page;
};

// One CTA per new token: warp 0 normalises, rotates and writes the latent row (16 latent elements a lane, the rotary part on
// its first lanes), the other warps rotate the query heads.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(128) latent_append_kernel(const LatentAppendArgs a) {
    const int64_t tok = blockIdx.x;
    const int64_t b = tok / a.S;
    const int j = (int)(tok - b * a.S);
    const int half = a.rope / 2, per = half / 8;  // lanes of a rotary row
    const float* cos = a.cos + tok * half;
    const float* sin = a.sin + tok * half;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int pid = 0, off = 0;
        if (!find_slot(a.table, a.table_stride, a.W, a.P, a.page, a.starts[b], j, a.counts ? a.counts[b] : a.S, b, pid, off)) return;
        const T* src = (const T*)a.a + b * a.a_b + j * a.a_s;
        float x[2][8] = {}, p[8] = {}, r[8] = {};
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = (lane + 32 * i) * 8;
            if (e < a.R) {
                Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + e), x[i]);
#pragma unroll
                for (int t = 0; t < 8; ++t) ss += x[i][t] * x[i][t];
            }
        }
        if (lane < per) {
            Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + a.R + lane * 8), p);
            Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + a.R + half + lane * 8), r);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float u = p[t], w = r[t], c = cos[lane * 8 + t], s = sin[lane * 8 + t];
                p[t] = u * c - w * s;
                r[t] = w * c + u * s;
            }
        }
        ss = warp_sum(ss);
        const float inv_rms = rsqrtf(ss / (float)a.R + a.eps);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int e = (lane + 32 * i) * 8;
            if (e < a.R) {
                float w[8];
                Vec8<T>::unpack(*reinterpret_cast<const uint4*>((const T*)a.w + e), w);
#pragma unroll
                for (int t = 0; t < 8; ++t) x[i][t] *= inv_rms * w[t];
            }
        }
        const int D = a.R + a.rope;
        if (E4M3) {
            float m = 0.f;
#pragma unroll
            for (int t = 0; t < 8; ++t)
                m = max_nan(m, max_nan(max_nan(fabsf(x[0][t]), fabsf(x[1][t])), max_nan(fabsf(p[t]), fabsf(r[t]))));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float scale = e4m3_scale(m), inv = __fdiv_rn(1.f, scale);
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                x[0][t] *= inv;
                x[1][t] *= inv;
                p[t] *= inv;
                r[t] *= inv;
            }
            uint8_t* dst = (uint8_t*)a.pages + pid * a.page_stride + (int64_t)off * D;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if ((lane + 32 * i) * 8 < a.R) *reinterpret_cast<uint2*>(dst + (lane + 32 * i) * 8) = pack_e4m3x8(x[i]);
            if (lane < per) {
                *reinterpret_cast<uint2*>(dst + a.R + lane * 8) = pack_e4m3x8(p);
                *reinterpret_cast<uint2*>(dst + a.R + half + lane * 8) = pack_e4m3x8(r);
            }
            if (lane == 0) a.scale[pid * a.scale_stride + off] = scale;
        } else {
            T* dst = (T*)a.pages + pid * a.page_stride + (int64_t)off * D;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if ((lane + 32 * i) * 8 < a.R) *reinterpret_cast<uint4*>(dst + (lane + 32 * i) * 8) = Vec8<T>::pack(x[i]);
            if (lane < per) {
                *reinterpret_cast<uint4*>(dst + a.R + lane * 8) = Vec8<T>::pack(p);
                *reinterpret_cast<uint4*>(dst + a.R + half + lane * 8) = Vec8<T>::pack(r);
            }
        }
        return;
    }
    for (int u = threadIdx.x - 32; u < a.H * per; u += 96) {
        const int h = u / per, lane = u - h * per;
        const T* src = (const T*)a.q + b * a.q_b + j * a.q_s + h * a.q_h;
        float p[8], r[8];
        Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + lane * 8), p);
        Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + half + lane * 8), r);
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const float x = p[t], y = r[t], c = cos[lane * 8 + t], s = sin[lane * 8 + t];
            p[t] = x * c - y * s;
            r[t] = y * c + x * s;
        }
        T* dst = (T*)a.q_out + (tok * a.H + h) * a.rope;
        *reinterpret_cast<uint4*>(dst + lane * 8) = Vec8<T>::pack(p);
        *reinterpret_cast<uint4*>(dst + half + lane * 8) = Vec8<T>::pack(r);
    }
}

struct ReadArgs {
    const void* pages;
    const float* scale;
    int64_t page_stride, scale_stride;
    void* out;  // [B, n, H, D]
    const int *table, *lengths;
    int64_t table_stride;
    int n, H, D, P, W, page;
};

// One thread per 8 elements of the output.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
    const int chunks = a.D / 8;
    const int64_t per_b = (int64_t)a.n * a.H * chunks;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= per_b) return;
    const int64_t b = blockIdx.y;
    const int64_t row = i / chunks;
    const int c = (int)(i - row * chunks);
    const int t = (int)(row / a.H), h = (int)(row - (int64_t)t * a.H);
    uint4 res = make_uint4(0, 0, 0, 0);
    const int len = min(a.lengths[b], a.W * a.page);
    if (t < len) {
        const int w = t / a.page, off = t - w * a.page;
        const int pid = a.table[b * a.table_stride + w];
        if (pid >= 0 && pid < a.P) {
            const int64_t at = pid * a.page_stride + ((int64_t)h * a.page + off) * a.D + c * 8;
            if (E4M3) {
                float f[8];
                unpack_e4m3x8(*reinterpret_cast<const uint2*>((const uint8_t*)a.pages + at), f);
                const float s = a.scale[pid * a.scale_stride + (int64_t)h * a.page + off];
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] *= s;
                res = Vec8<T>::pack(f);
            } else {
                res = *reinterpret_cast<const uint4*>((const T*)a.pages + at);
            }
        }
    }
    *reinterpret_cast<uint4*>((T*)a.out + (b * per_b + i) * 8) = res;
}

static bool kernel_dtype(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

static void check_cos_sin(const char* op, const at::Tensor& cos, const at::Tensor& sin, int64_t B, int64_t S, int64_t half,
                          const at::Tensor& x) {
    ATB_ARG(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.dim() == 3 && sin.dim() == 3 &&
                cos.size(0) == B && cos.size(1) == S && cos.size(2) == half && sin.sizes() == cos.sizes(),
            op, ": cos and sin must be fp32 [batch, new tokens, rotary width / 2]");
    ATB_ARG(cos.device() == x.device() && sin.device() == x.device(), op, ": all tensors must be on one device");
}

template <typename T, bool E4M3>
static void launch_append(const AppendArgs& a, int64_t tokens, cudaStream_t st) {
    const int lanes = a.D / 16;
    const dim3 grid((unsigned)tokens);
    if (lanes <= 1) append_kernel<T, E4M3, 1><<<grid, 256, 0, st>>>(a);
    else if (lanes <= 2) append_kernel<T, E4M3, 2><<<grid, 256, 0, st>>>(a);
    else if (lanes <= 4) append_kernel<T, E4M3, 4><<<grid, 256, 0, st>>>(a);
    else if (lanes <= 8) append_kernel<T, E4M3, 8><<<grid, 256, 0, st>>>(a);
    else append_kernel<T, E4M3, 16><<<grid, 256, 0, st>>>(a);
}

}  // namespace paged

using namespace paged;

at::Tensor paged_kv_append(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& cos,
                           const at::Tensor& sin, at::Tensor k_pages, at::Tensor v_pages, const at::Tensor& table,
                           const at::Tensor& starts, const c10::optional<at::Tensor>& counts,
                           const c10::optional<at::Tensor>& k_scale, const c10::optional<at::Tensor>& v_scale) {
    const char* op = "paged_kv_append";
    ATB_ARG(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, op, ": q, k and v must be [batch, new tokens, heads, dim]");
    const int64_t B = q.size(0), S = q.size(1), Hq = q.size(2), D = q.size(3), Hkv = k.size(2);
    ATB_ARG(k.size(0) == B && k.size(1) == S && k.size(3) == D && v.sizes() == k.sizes(), op, ": q, k and v differ in shape");
    ATB_ARG(kernel_dtype(q) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(), op,
            ": q, k and v must be bf16 or fp16, all of one type");
    ATB_ARG(D % 16 == 0 && D <= 256 && D > 0, op, ": dim must be a multiple of 16 up to 256");
    ATB_ARG(k.device() == q.device() && v.device() == q.device(), op, ": all tensors must be on one device");
    check_cos_sin(op, cos, sin, B, S, D / 2, q);
    check_pages(op, k_pages, k_scale, q);
    check_pages(op, v_pages, v_scale, q);
    ATB_ARG(k_pages.sizes() == v_pages.sizes() && k_pages.scalar_type() == v_pages.scalar_type(), op, ": k_pages and v_pages differ");
    ATB_ARG(k_pages.size(1) == Hkv && k_pages.size(3) == D, op, ": the cache has other heads or another dim than k");
    ATB_ARG(is_e4m3(k_pages) || k_pages.scalar_type() == q.scalar_type(), op, ": the cache must have the inputs' type or be e4m3");
    check_table(op, table, starts, counts, k_pages, B);
    ATB_ARG(B * S < (int64_t(1) << 31), op, ": too many tokens");
    const c10::cuda::CUDAGuard guard(q.device());
    at::Tensor out = at::empty({B, S, Hq, D}, q.options());
    if (B * S == 0) return out;
    const at::Tensor qc = rows16(q), kc = rows16(k), vc = rows16(v), cc = rows16(cos.contiguous()), sc = rows16(sin.contiguous());
    AppendArgs a;
    a.q = qc.data_ptr(); a.k = kc.data_ptr(); a.v = vc.data_ptr();
    a.q_b = qc.stride(0); a.q_s = qc.stride(1); a.q_h = qc.stride(2);
    a.k_b = kc.stride(0); a.k_s = kc.stride(1); a.k_h = kc.stride(2);
    a.v_b = vc.stride(0); a.v_s = vc.stride(1); a.v_h = vc.stride(2);
    a.cos = cc.data_ptr<float>(); a.sin = sc.data_ptr<float>();
    a.q_out = out.data_ptr();
    a.k_pages = k_pages.data_ptr(); a.v_pages = v_pages.data_ptr();
    a.k_scale = ptr<float>(k_scale); a.v_scale = ptr<float>(v_scale);
    a.k_page = k_pages.stride(0); a.v_page = v_pages.stride(0);
    a.ks_page = k_scale.has_value() ? k_scale->stride(0) : 0; a.vs_page = v_scale.has_value() ? v_scale->stride(0) : 0;
    a.table = table.data_ptr<int>(); a.starts = starts.data_ptr<int>(); a.counts = ptr<int>(counts);
    a.table_stride = table.stride(0);
    a.S = (int)S; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = (int)D; a.P = (int)k_pages.size(0); a.W = (int)table.size(1);
    a.page = (int)k_pages.size(2);
    const bool f8 = is_e4m3(k_pages);
    cudaStream_t st = current_stream();
    if (q.scalar_type() == at::kBFloat16) f8 ? launch_append<bf16, true>(a, B * S, st) : launch_append<bf16, false>(a, B * S, st);
    else f8 ? launch_append<__half, true>(a, B * S, st) : launch_append<__half, false>(a, B * S, st);
    ATB_LAUNCH_CHECK();
    return out;
}

at::Tensor paged_latent_append(const at::Tensor& q_pe, const at::Tensor& kv_a, const at::Tensor& weight, double eps,
                               const at::Tensor& cos, const at::Tensor& sin, at::Tensor pages, const at::Tensor& table,
                               const at::Tensor& starts, const c10::optional<at::Tensor>& counts,
                               const c10::optional<at::Tensor>& scale) {
    const char* op = "paged_latent_append";
    ATB_ARG(q_pe.dim() == 4 && kv_a.dim() == 3, op, ": q_pe must be [batch, new tokens, heads, rotary] and kv_a [batch, new tokens, latent + rotary]");
    const int64_t B = q_pe.size(0), S = q_pe.size(1), H = q_pe.size(2), rope = q_pe.size(3), R = weight.numel();
    ATB_ARG(weight.dim() == 1 && kv_a.size(0) == B && kv_a.size(1) == S && kv_a.size(2) == R + rope, op,
            ": q_pe, kv_a and norm_weight differ in shape");
    ATB_ARG(kernel_dtype(q_pe) && kv_a.scalar_type() == q_pe.scalar_type() && weight.scalar_type() == q_pe.scalar_type(), op,
            ": q_pe, kv_a and norm_weight must be bf16 or fp16, all of one type");
    ATB_ARG(R % 16 == 0 && R > 0 && R <= 512 && rope % 16 == 0 && rope > 0 && rope <= 64, op,
            ": the latent must be a multiple of 16 up to 512, the rotary part one up to 64");
    ATB_ARG(kv_a.device() == q_pe.device() && weight.device() == q_pe.device(), op, ": all tensors must be on one device");
    check_cos_sin(op, cos, sin, B, S, rope / 2, q_pe);
    check_pages(op, pages, scale, q_pe);
    ATB_ARG(pages.size(1) == 1 && pages.size(3) == R + rope, op, ": a latent cache is [pages, 1, page, latent + rotary]");
    ATB_ARG(is_e4m3(pages) || pages.scalar_type() == q_pe.scalar_type(), op, ": the cache must have the inputs' type or be e4m3");
    check_table(op, table, starts, counts, pages, B);
    ATB_ARG(B * S < (int64_t(1) << 31), op, ": too many tokens");
    const c10::cuda::CUDAGuard guard(q_pe.device());
    at::Tensor out = at::empty({B, S, H, rope}, q_pe.options());
    if (B * S == 0) return out;
    const at::Tensor qc = rows16(q_pe), ac = rows16(kv_a), wc = rows16(weight), cc = cos.contiguous(), sc = sin.contiguous();
    LatentAppendArgs a;
    a.q = qc.data_ptr(); a.a = ac.data_ptr(); a.w = wc.data_ptr();
    a.q_b = qc.stride(0); a.q_s = qc.stride(1); a.q_h = qc.stride(2); a.a_b = ac.stride(0); a.a_s = ac.stride(1);
    a.cos = cc.data_ptr<float>(); a.sin = sc.data_ptr<float>();
    a.q_out = out.data_ptr();
    a.pages = pages.data_ptr(); a.scale = ptr<float>(scale);
    a.page_stride = pages.stride(0); a.scale_stride = scale.has_value() ? scale->stride(0) : 0;
    a.table = table.data_ptr<int>(); a.starts = starts.data_ptr<int>(); a.counts = ptr<int>(counts);
    a.table_stride = table.stride(0);
    a.eps = (float)eps;
    a.S = (int)S; a.H = (int)H; a.R = (int)R; a.rope = (int)rope; a.P = (int)pages.size(0); a.W = (int)table.size(1);
    a.page = (int)pages.size(2);
    const bool f8 = is_e4m3(pages);
    cudaStream_t st = current_stream();
    const dim3 grid((unsigned)(B * S));
    if (q_pe.scalar_type() == at::kBFloat16) {
        if (f8) latent_append_kernel<bf16, true><<<grid, 128, 0, st>>>(a);
        else latent_append_kernel<bf16, false><<<grid, 128, 0, st>>>(a);
    } else {
        if (f8) latent_append_kernel<__half, true><<<grid, 128, 0, st>>>(a);
        else latent_append_kernel<__half, false><<<grid, 128, 0, st>>>(a);
    }
    ATB_LAUNCH_CHECK();
    return out;
}

at::Tensor paged_read(const at::Tensor& pages, const at::Tensor& table, const at::Tensor& lengths, int64_t max_length,
                      const c10::optional<at::Tensor>& scale, at::ScalarType dtype) {
    const char* op = "paged_kv_read";
    ATB_ARG(table.dim() == 2, op, ": page_table must be int32 [batch, pages]");
    const int64_t B = table.size(0);
    check_pages(op, pages, scale, pages);
    check_table(op, table, lengths, c10::nullopt, pages, B);
    const int64_t H = pages.size(1), D = pages.size(3);
    ATB_ARG(D % 16 == 0 && D > 0, op, ": dim must be a multiple of 16");
    ATB_ARG(dtype == at::kBFloat16 || dtype == at::kHalf, op, ": the result must be bf16 or fp16");
    ATB_ARG(is_e4m3(pages) || pages.scalar_type() == dtype, op, ": the cache must have the result's type or be e4m3");
    ATB_ARG(max_length >= 0 && max_length < (int64_t(1) << 31), op, ": max_length must be 0 or more");
    ATB_ARG(B <= 65535, op, ": too many sequences");
    const c10::cuda::CUDAGuard guard(pages.device());
    at::Tensor out = at::empty({B, max_length, H, D}, pages.options().dtype(dtype));
    if (out.numel() == 0) return out;
    ReadArgs a;
    a.pages = pages.data_ptr(); a.scale = ptr<float>(scale);
    a.page_stride = pages.stride(0); a.scale_stride = scale.has_value() ? scale->stride(0) : 0;
    a.out = out.data_ptr();
    a.table = table.data_ptr<int>(); a.lengths = lengths.data_ptr<int>(); a.table_stride = table.stride(0);
    a.n = (int)max_length; a.H = (int)H; a.D = (int)D; a.P = (int)pages.size(0); a.W = (int)table.size(1); a.page = (int)pages.size(2);
    const int64_t blocks = ceil_div(max_length * H * (D / 8), 256);
    ATB_ARG(blocks < (int64_t(1) << 31), op, ": the result is too large");
    const dim3 grid((unsigned)blocks, (unsigned)B);
    cudaStream_t st = current_stream();
    if (dtype == at::kBFloat16) {
        if (is_e4m3(pages)) read_kernel<bf16, true><<<grid, 256, 0, st>>>(a);
        else read_kernel<bf16, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (is_e4m3(pages)) read_kernel<__half, true><<<grid, 256, 0, st>>>(a);
        else read_kernel<__half, false><<<grid, 256, 0, st>>>(a);
    }
    ATB_LAUNCH_CHECK();
    return out;
}

}  // namespace atb
