// SPDX-License-Identifier: Apache-2.0
// Writing and reading the paged generation cache: rotation of queries and keys fused with the write of keys and values
// (plain or e4m3), the same for latent rows with their RMS norm, and the read-back into dense tensors.
// All of it is bound by memory traffic: every input is read once and every output written once, in 16-byte accesses.
#include <algorithm>
#include <tuple>

#include "paged_common.cuh"

namespace atb {
namespace paged {

// Where the new token (b, j) goes: page id and offset; a page id of -1 when it is not written.
__device__ __forceinline__ int find_slot(const int* __restrict__ table, int64_t table_stride, int W, int P, int page, int start,
                                         int j, int count, int64_t b, int& off) {
    off = 0;
    if (j >= count || start < 0) return -1;
    const int64_t pos = (int64_t)start + j;
    if (pos >= (int64_t)W * page) return -1;
    const int w = (int)pos / page;
    off = (int)pos - w * page;
    const int pid = table[b * table_stride + w];
    return pid < P ? max(pid, -1) : -1;
}

__device__ __forceinline__ void load8(const float* src, float (&f)[8]) {
    const float4 x = reinterpret_cast<const float4*>(src)[0], y = reinterpret_cast<const float4*>(src)[1];
    f[0] = x.x; f[1] = x.y; f[2] = x.z; f[3] = x.w; f[4] = y.x; f[5] = y.y; f[6] = y.z; f[7] = y.w;
}

// A rotation of the pairs (x, y), products and sums rounded one by one: contracted, a value next to a rounding border would be
// stored as its neighbour, and an 8-bit row would hold other bytes than the reference writes for the same input.
__device__ __forceinline__ void rotate8(float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float u = x[i], w = y[i];
        x[i] = __fsub_rn(__fmul_rn(u, c[i]), __fmul_rn(w, s[i]));
        y[i] = __fadd_rn(__fmul_rn(w, c[i]), __fmul_rn(u, s[i]));
    }
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
// sin of a lane are loaded once and serve all heads of the token.  The next row is on its way while one is worked on, and the
// place in the cache is looked up behind the first loads.  Few tokens get a wide CTA (all rows at once: latency counts),
// many get narrow ones, 16 to an SM, whose fixed chain of loads (lengths, page, cos / sin) overlaps.
// Measured: one token of 32 + 16 heads 2.6 us (launch); 12 prompts of up to 1511 tokens, 28 + 8 heads, into an 8-bit cache (301
// MB) 52 us, 90 % of a plain copy's rate, and as they are (311 MB) 52 us, 93 %.
template <typename T, bool E4M3, int LPR>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a) {
    const int64_t tok = blockIdx.x;
    const int64_t b = tok / a.S;
    const int j = (int)(tok - b * a.S);
    const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, groups = blockDim.x / LPR;
    const int half = a.D / 2;
    const bool active = lane * 8 < half;
    const int start = a.starts[b], count = a.counts ? a.counts[b] : a.S;
    const int rows = j < count ? a.Hq + 2 * a.Hkv : a.Hq;
    auto load = [&](int r, uint4& lo, uint4& hi) {
        lo = hi = make_uint4(0, 0, 0, 0);
        if (r >= rows || !active) return;
        const T* src;
        if (r < a.Hq) src = (const T*)a.q + b * a.q_b + j * a.q_s + r * a.q_h;
        else if (r < a.Hq + a.Hkv) src = (const T*)a.k + b * a.k_b + j * a.k_s + (r - a.Hq) * a.k_h;
        else src = (const T*)a.v + b * a.v_b + j * a.v_s + (r - a.Hq - a.Hkv) * a.v_h;
        lo = *reinterpret_cast<const uint4*>(src + lane * 8);
        hi = *reinterpret_cast<const uint4*>(src + half + lane * 8);
    };
    uint4 next_lo, next_hi;
    load(group, next_lo, next_hi);
    float c[8], s[8];
    if (active) {
        load8(a.cos + tok * half + lane * 8, c);
        load8(a.sin + tok * half + lane * 8, s);
    }
    int off;
    const int pid = find_slot(a.table, a.table_stride, a.W, a.P, a.page, start, j, count, b, off);
    // every lane of a warp takes the same number of rounds, so the shuffles below are complete
    for (int r0 = 0; r0 < rows; r0 += groups) {
        const int r = r0 + group;
        const bool mine = r < rows && active;
        const int kind = r < a.Hq ? 0 : (r < a.Hq + a.Hkv ? 1 : 2);
        float x[8], y[8];
        Vec8<T>::unpack(next_lo, x);
        Vec8<T>::unpack(next_hi, y);
        load(r + groups, next_lo, next_hi);
        if (mine && kind != 2) rotate8(x, y, c, s);
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
        if (pid < 0) continue;
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
// its first lanes), the others (enough for two rounds over all heads) rotate the queries.  Measured: 96 tokens 3.0 us; 8 prompts
// of up to 2048 tokens (97 MB) 21 us, 71 % of a plain copy's rate, into 8-bit rows (90 MB) 22 us, 63 %: a token's chain of lengths,
// row or page, weight and write, with nothing of the next token on its way.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) latent_append_kernel(const LatentAppendArgs a) {
    const int64_t tok = blockIdx.x;
    const int64_t b = tok / a.S;
    const int j = (int)(tok - b * a.S);
    const int half = a.rope / 2, per = half / 8;  // lanes of a rotary row
    const float* cos = a.cos + tok * half;
    const float* sin = a.sin + tok * half;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const int start = a.starts[b], count = a.counts ? a.counts[b] : a.S;
        if (j >= count || start < 0) return;
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
        int off;
        const int pid = find_slot(a.table, a.table_stride, a.W, a.P, a.page, start, j, count, b, off);
        if (lane < per) {
            Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + a.R + lane * 8), p);
            Vec8<T>::unpack(*reinterpret_cast<const uint4*>(src + a.R + half + lane * 8), r);
            float c[8], s[8];
            load8(cos + lane * 8, c);
            load8(sin + lane * 8, s);
            rotate8(p, r, c, s);
        }
        if (pid < 0) return;  // the whole warp
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
    // two pieces of 16 elements a round, loaded before either is worked on
    const int units = a.H * per, step = blockDim.x - 32;
    for (int u0 = threadIdx.x - 32; u0 < units; u0 += 2 * step) {
        uint4 lo[2], hi[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int u = u0 + x * step, h = u / per, lane = u - h * per;
            if (u >= units) continue;
            const T* src = (const T*)a.q + b * a.q_b + j * a.q_s + h * a.q_h;
            lo[x] = *reinterpret_cast<const uint4*>(src + lane * 8);
            hi[x] = *reinterpret_cast<const uint4*>(src + half + lane * 8);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int u = u0 + x * step, h = u / per, lane = u - h * per;
            if (u >= units) continue;
            float p[8], r[8], c[8], s[8];
            load8(cos + lane * 8, c);
            load8(sin + lane * 8, s);
            Vec8<T>::unpack(lo[x], p);
            Vec8<T>::unpack(hi[x], r);
            rotate8(p, r, c, s);
            T* dst = (T*)a.q_out + (tok * a.H + h) * a.rope;
            *reinterpret_cast<uint4*>(dst + lane * 8) = Vec8<T>::pack(p);
            *reinterpret_cast<uint4*>(dst + half + lane * 8) = Vec8<T>::pack(r);
        }
    }
}

struct ReadArgs {
    const void* pages[2];  // keys, values
    const float* scale[2];
    int64_t page_stride[2], scale_stride[2];
    void* out[2];  // [B, n, H, D]
    const int *table, *lengths;
    int64_t table_stride;
    int n, H, D, P, W, page;
    uint32_t magic;  // 2^32 / (D / 8), rounded up
};

// One CTA per kReadRows rows (position, head) of one sequence's keys or values.  The places of the rows are looked up once, into
// shared memory; then every thread moves 16-byte pieces of the result, four on their way at a time.  Measured: 16 sequences of
// up to 16000 8-bit latent rows (392 MB) 67 us, 91 % of a plain copy's rate, and plain ones (488 MB) 80 us, 94 %.
constexpr int kReadRows = 64, kReadDim = 2048;  // 64 rows of at most 256 chunks
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs a) {
    __shared__ int64_t s_at[kReadRows];
    __shared__ float s_scale[kReadRows];
    const int chunks = a.D / 8, z = blockIdx.z;
    const int64_t b = blockIdx.y, rows = (int64_t)a.n * a.H, row0 = (int64_t)blockIdx.x * kReadRows;
    const int here = (int)min((int64_t)kReadRows, rows - row0);
    if (threadIdx.x < here) {
        const int64_t row = row0 + threadIdx.x;
        const int t = (int)(row / a.H), h = (int)(row - (int64_t)t * a.H);
        int64_t at = -1;
        float scale = 0.f;
        if (t < min(a.lengths[b], a.W * a.page)) {
            const int w = t / a.page, off = t - w * a.page;
            const int pid = a.table[b * a.table_stride + w];
            if (pid >= 0 && pid < a.P) {
                at = pid * a.page_stride[z] + ((int64_t)h * a.page + off) * a.D;
                if (E4M3) scale = a.scale[z][pid * a.scale_stride[z] + (int64_t)h * a.page + off];
            }
        }
        s_at[threadIdx.x] = at;
        s_scale[threadIdx.x] = scale;
    }
    __syncthreads();
    uint4* out = reinterpret_cast<uint4*>((T*)a.out[z] + (b * rows + row0) * a.D);
    const int total = here * chunks;
    for (int i0 = threadIdx.x; i0 < total; i0 += 4 * 256) {
        uint4 v[4];
        float s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + k * 256;
            v[k] = make_uint4(0, 0, 0, 0);
            s[k] = 0.f;
            if (i >= total) continue;
            const int r = (int)__umulhi((uint32_t)i, a.magic);  // i / chunks: exact for i < 2^16
            const int64_t at = s_at[r];
            if (at < 0) continue;
            const int64_t e = at + (i - r * chunks) * 8;
            if (E4M3) {
                const uint2 u = *reinterpret_cast<const uint2*>((const uint8_t*)a.pages[z] + e);
                v[k].x = u.x;
                v[k].y = u.y;
                s[k] = s_scale[r];
            } else {
                v[k] = *reinterpret_cast<const uint4*>((const T*)a.pages[z] + e);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = i0 + k * 256;
            if (i >= total) continue;
            if (E4M3) {
                float f[8];
                unpack_e4m3x8(make_uint2(v[k].x, v[k].y), f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] *= s[k];
                v[k] = Vec8<T>::pack(f);
            }
            out[i] = v[k];
        }
    }
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
    // narrow CTAs from about three resident sets of wide ones on (12 prompts of up to 1511 tokens, 301 MB: 64 threads 51.3 us,
    // 128 56.3 us, 256 76.4 us; one token: 256 threads)
    const int threads = tokens > 1000 ? 64 : 256;
    if (lanes <= 1) append_kernel<T, E4M3, 1><<<grid, threads, 0, st>>>(a);
    else if (lanes <= 2) append_kernel<T, E4M3, 2><<<grid, threads, 0, st>>>(a);
    else if (lanes <= 4) append_kernel<T, E4M3, 4><<<grid, threads, 0, st>>>(a);
    else if (lanes <= 8) append_kernel<T, E4M3, 8><<<grid, threads, 0, st>>>(a);
    else append_kernel<T, E4M3, 16><<<grid, threads, 0, st>>>(a);
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
    const at::Tensor qc = rows16(q_pe), ac = rows16(kv_a), wc = rows16(weight), cc = rows16(cos.contiguous()), sc = rows16(sin.contiguous());
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
    const unsigned threads = 32 + 32 * (unsigned)std::min<int64_t>(7, std::max<int64_t>(1, ceil_div(H * (rope / 16), 64)));
    if (q_pe.scalar_type() == at::kBFloat16) {
        if (f8) latent_append_kernel<bf16, true><<<grid, threads, 0, st>>>(a);
        else latent_append_kernel<bf16, false><<<grid, threads, 0, st>>>(a);
    } else {
        if (f8) latent_append_kernel<__half, true><<<grid, threads, 0, st>>>(a);
        else latent_append_kernel<__half, false><<<grid, threads, 0, st>>>(a);
    }
    ATB_LAUNCH_CHECK();
    return out;
}

std::tuple<at::Tensor, at::Tensor> paged_read(const at::Tensor& k_pages, const c10::optional<at::Tensor>& v_pages, const at::Tensor& table,
                                              const at::Tensor& lengths, int64_t max_length, const c10::optional<at::Tensor>& k_scale,
                                              const c10::optional<at::Tensor>& v_scale, at::ScalarType dtype) {
    const char* op = "paged_kv_read";
    ATB_ARG(table.dim() == 2, op, ": page_table must be int32 [batch, pages]");
    const int64_t B = table.size(0);
    check_pages(op, k_pages, k_scale, k_pages);
    check_table(op, table, lengths, c10::nullopt, k_pages, B);
    const int64_t H = k_pages.size(1), D = k_pages.size(3);
    ATB_ARG(D % 16 == 0 && D > 0 && D <= kReadDim, op, ": dim must be a multiple of 16 up to ", kReadDim);
    ATB_ARG(dtype == at::kBFloat16 || dtype == at::kHalf, op, ": the result must be bf16 or fp16");
    ATB_ARG(is_e4m3(k_pages) || k_pages.scalar_type() == dtype, op, ": the cache must have the result's type or be e4m3");
    if (v_pages.has_value()) {
        check_pages(op, *v_pages, v_scale, k_pages);
        ATB_ARG(v_pages->sizes() == k_pages.sizes() && v_pages->scalar_type() == k_pages.scalar_type(), op, ": k_pages and v_pages differ");
    }
    ATB_ARG(max_length >= 0 && max_length < (int64_t(1) << 31), op, ": max_length must be 0 or more");
    ATB_ARG(B <= 65535, op, ": too many sequences");
    const c10::cuda::CUDAGuard guard(k_pages.device());
    const int tensors = v_pages.has_value() ? 2 : 1;
    at::Tensor k = at::empty({B, max_length, H, D}, k_pages.options().dtype(dtype));
    at::Tensor v = at::empty({tensors == 2 ? B : 0, max_length, H, D}, k_pages.options().dtype(dtype));
    if (k.numel() == 0) return {k, v};
    ReadArgs a;
    a.pages[0] = k_pages.data_ptr(); a.scale[0] = ptr<float>(k_scale);
    a.page_stride[0] = k_pages.stride(0); a.scale_stride[0] = k_scale.has_value() ? k_scale->stride(0) : 0;
    a.out[0] = k.data_ptr();
    a.pages[1] = tensors == 2 ? v_pages->data_ptr() : nullptr; a.scale[1] = ptr<float>(v_scale);
    a.page_stride[1] = tensors == 2 ? v_pages->stride(0) : 0; a.scale_stride[1] = v_scale.has_value() ? v_scale->stride(0) : 0;
    a.out[1] = v.data_ptr();
    a.table = table.data_ptr<int>(); a.lengths = lengths.data_ptr<int>(); a.table_stride = table.stride(0);
    a.n = (int)max_length; a.H = (int)H; a.D = (int)D; a.P = (int)k_pages.size(0); a.W = (int)table.size(1); a.page = (int)k_pages.size(2);
    a.magic = (uint32_t)(((uint64_t(1) << 32) + D / 8 - 1) / (D / 8));
    const int64_t blocks = ceil_div(max_length * H, kReadRows);
    ATB_ARG(blocks < (int64_t(1) << 31), op, ": the result is too large");
    const dim3 grid((unsigned)blocks, (unsigned)B, (unsigned)tensors);
    cudaStream_t st = current_stream();
    if (dtype == at::kBFloat16) {
        if (is_e4m3(k_pages)) read_kernel<bf16, true><<<grid, 256, 0, st>>>(a);
        else read_kernel<bf16, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (is_e4m3(k_pages)) read_kernel<__half, true><<<grid, 256, 0, st>>>(a);
        else read_kernel<__half, false><<<grid, 256, 0, st>>>(a);
    }
    ATB_LAUNCH_CHECK();
    return {k, v};
}

}  // namespace atb
