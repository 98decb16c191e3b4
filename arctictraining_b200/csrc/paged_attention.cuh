// SPDX-License-Identifier: Apache-2.0
// What the attention kernels over the paged generation cache share: arguments, division of the work, matrix instructions and
// the joining of pieces.
//
// Query j of a sequence stands at position p = starts + j and sees the cached positions max(0, p - window + 1) .. p:
// o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m), s_t = scale q.k_t, in one pass over the keys with the running maximum m.
// The latent form has one key row [latent | rotary] for all heads and the latent itself as value.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

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
    // division into items (set by the launch): empty rounds before an item, value columns of an item and items beside one
    // another that share the columns, tiles of query rows of a token where tiles do not cross tokens (else 0)
    int lead, cols, halves, token_tiles;
};

// The query rows (token, head of the group) of an item: cache head, part of the columns, first row, number of rows.
__device__ __forceinline__ void item_rows(const AttnArgs& a, int item, int rows, int& h, int& half, int& row0, int& n) {
    const int G = a.Hq / a.Hkv, t = item / a.halves;
    half = item - t * a.halves;
    if (a.token_tiles) {
        const int j = t / a.token_tiles, tile = t - j * a.token_tiles;
        h = 0;
        row0 = j * G + tile * rows;
        n = min(rows, G - tile * rows);
    } else {
        const int M = a.S * G, tiles = (M + rows - 1) / rows;
        h = t / tiles;
        row0 = (t - h * tiles) * rows;
        n = min(rows, M - row0);
    }
}

// ---- schedule ---------------------------------------------------------------------------------------------------------
// Work is counted in rounds of `NK` keys of one item (sequence, cache head, tile of query rows).  The rounds of all items
// stand in one line, each item's behind `lead` empty ones that stand for what an item costs besides its keys (its queries,
// the pipeline's filling, the result: 2 to 3 us for grouped heads, where a round takes 1.5 to 2 us), and every CTA takes an
// equal piece of the line, so a batch of very different lengths loads all SMs alike and a single long sequence is spread over
// all of them (without the empty rounds the ragged batch below took 88 us, 15 of them for the CTA with most items).  A CTA that covers an item alone writes the result; otherwise it
// leaves (maximum, sum, weighted values) of its piece in the workspace, and the join kernel adds the pieces in their
// order.  No atomics: the same inputs give the same bits.
struct Range {  // the cached positions that the queries of one sequence see
    int start, total, low, first, rounds;  // positions [low, total); counted from `first`, a multiple of NK
};
__device__ __forceinline__ Range seq_range(const AttnArgs& a, int b, int NK) {
    Range r;
    r.start = a.starts[b];
    const int count = a.counts ? max(0, min(a.counts[b], a.S)) : a.S;
    const int64_t cap = (int64_t)a.W * a.page, end = (int64_t)r.start + count;
    r.total = count == 0 ? 0 : (int)max((int64_t)0, min(end, cap));
    r.low = a.window > 0 ? (int)max((int64_t)0, min((int64_t)r.start + 1 - a.window, (int64_t)r.total)) : 0;
    r.first = r.low / NK * NK;
    r.rounds = a.lead + max(1, (r.total - r.first + NK - 1) / NK);  // a sequence that sees nothing has one round, fully masked
    return r;
}

// How `all` rounds are divided: the first `rest` CTAs take one more than the others.  (32-bit: the host bounds the line.)
struct Pieces {
    int share, rest;
    __device__ __forceinline__ Pieces(int all, int ctas) : share(all / ctas), rest(all - all / ctas * ctas) {}
    __device__ __forceinline__ int begin(int cta) const { return cta * share + min(cta, rest); }
    __device__ __forceinline__ int cta_of(int round) const {
        const int wide = rest * (share + 1);
        return round < wide ? round / (share + 1) : rest + (round - wide) / max(share, 1);
    }
};

// The line's division, and of CTA `cta`'s piece [at, to) the sequence that holds its first round (a sequence has `per` items)
// and that sequence's first round.
template <int THREADS>
__device__ __forceinline__ Pieces find_piece(const AttnArgs& a, int B, int NK, int per, int ctas, int cta, int& at, int& to, int& b_out,
                                             int& line, int* scratch) {
    // thread i looks at sequences [i n, (i + 1) n)
    const int n = (B + THREADS - 1) / THREADS, b0 = threadIdx.x * n, b1 = min(B, b0 + n);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += seq_range(a, b, NK).rounds;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) base += scratch[w];
        all += scratch[w];
    }
    const Pieces pieces(all * per, ctas);
    at = pieces.begin(cta);
    to = pieces.begin(cta + 1);
    int lo = (base + incl - mine) * per;
    if (at < to && at >= lo && at < lo + mine * per) {
        int b = b0;
        while (true) {
            const int r = seq_range(a, b, NK).rounds * per;
            if (at < lo + r) break;
            lo += r;
            ++b;
        }
        scratch[THREADS / 32] = b;
        scratch[THREADS / 32 + 1] = lo;
    }
    __syncthreads();
    b_out = scratch[THREADS / 32];
    line = scratch[THREADS / 32 + 1];
    return pieces;
}

// What the join kernel has to do at the begin of CTA k's piece: nothing, or join the `n` pieces of the item that CTA k - 1
// began and this CTA goes on with; x: sequence, y: item, z: n, w: the first piece is its CTA's first or second.
__device__ __forceinline__ int4 join_job(const AttnArgs& a, const Pieces& pieces, int cta, int at, int to, int b, int line, const Range& rg) {
    if (cta == 0 || at >= to) return make_int4(0, 0, 0, 0);
    const int item = (at - line) / rg.rounds, s = line + item * rg.rounds;
    if (pieces.cta_of(s + a.lead) != cta - 1) return make_int4(0, 0, 0, 0);
    return make_int4(b, item, pieces.cta_of(s + rg.rounds - 1) - cta + 2, pieces.begin(cta - 1) >= s ? 0 : 1);
}

// ---- tensor-core pieces -----------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// c += a b for a 16 x 16, b 16 x 8 of 16-bit elements, fp32 sums
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<bf16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<bf16>(float lo, float hi) {
    const bf162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<bf16>(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const bf162*>(&u)); }
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool full) {  // asynchronous; zeros where not `full`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(full ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool full) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(full ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// whether some value of the step is an infinity or a NaN (all bits of its exponent set)
template <typename P, int N, int KP, int CPR, typename F>
__device__ __forceinline__ bool values_not_finite(F&& load) {
    constexpr uint32_t e = std::is_same<P, bf16>::value ? 0x7f80u : 0x7c00u;
    bool bad = false;
#pragma unroll 1
    for (int kp = 0; kp < KP; ++kp)
#pragma unroll
        for (int k = 0; k < CPR; k += 2) {
            uint32_t v[N];
            load(kp, k, v);
#pragma unroll
            for (int x = 0; x < N; ++x) bad = bad || (v[x] & e) == e || ((v[x] >> 16) & e) == e;
        }
    return __any_sync(0xffffffffu, bad);
}

constexpr float kLog2e = 1.4426950408889634f;

constexpr int kMaxCtas = 1024;
struct JobList {  // in shared memory
    int4 jobs[kMaxCtas];
    int first[kMaxCtas], place[32], most;  // the CTA that began the item; most pieces of one
};
// All blocks of a joining kernel (128 threads) wait for the attention kernel, launched before, and gather its jobs in the
// order of their CTAs.  Returns their number.  (The pointers of such kernels are not declared free of aliases: loads that are
// known to be invariant may be moved ahead of the wait.)
__device__ __forceinline__ int gather_jobs(JobList& list, int ctas, const int4* jobs) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) list.most = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int4 mine[kMaxCtas / 128];
#pragma unroll
    for (int x = 0; x < kMaxCtas / 128; ++x) {
        const int k = threadIdx.x + 128 * x;
        mine[x] = k < ctas ? jobs[k] : make_int4(0, 0, 0, 0);
    }
    static_assert(kMaxCtas / 128 * 4 <= 32, "one lane per warp and round");
    uint32_t has[kMaxCtas / 128];
#pragma unroll
    for (int x = 0; x < kMaxCtas / 128; ++x) {
        has[x] = __ballot_sync(0xffffffffu, mine[x].z > 0);
        if (lane == 0) list.place[x * 4 + warp] = __popc(has[x]);
    }
    __syncthreads();
    int upto = list.place[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
    }
    const int n_jobs = __shfl_sync(0xffffffffu, upto, 31);
#pragma unroll
    for (int x = 0; x < kMaxCtas / 128; ++x) {
        const int base = __shfl_sync(0xffffffffu, upto, x * 4 + warp) - __popc(has[x]);
        if (mine[x].z > 0) {
            const int at = base + __popc(has[x] & ((1u << lane) - 1));
            list.jobs[at] = mine[x];
            list.first[at] = threadIdx.x + 128 * x - 1;
            atomicMax(&list.most, mine[x].z);
        }
    }
    __syncthreads();
    return n_jobs;
}

// Adds the pieces of an item that several CTAs of the attention kernel worked on, in their order along the keys.  Such an item
// lies across the begin of some CTA's piece; the attention kernel left a job there.  Every block gathers the jobs, all in the
// same order, and the blocks share out (job, query row, 128 columns): a warp each where the items have few pieces, a block
// each, its warps taking pieces in turn, where some item has many.
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const AttnArgs a, int rows, int ctas, const int4* jobs, const float* part_ml,
                                                   const float* part_o) {
    __shared__ JobList list;
    __shared__ float2 s_ml[kMaxCtas];
    __shared__ float s_red[2][4];
    __shared__ float4 s_o[128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n_jobs = gather_jobs(list, ctas, jobs);
    const int G = a.Hq / a.Hkv, M = a.S * G;
    const int used = min(rows, a.token_tiles ? G : M), slices = (a.cols / 4 + 31) / 32;
    const int total = n_jobs * used * slices;
    const bool wide = list.most > 8;  // a block for each unit
    for (int u = wide ? blockIdx.x : blockIdx.x * 4 + warp; u < total; u += wide ? gridDim.x : gridDim.x * 4) {
        const int col = (u % slices) * 128 + lane * 4, rest = u / slices;
        const int r = rest % used, jb = rest / used;
        const int4 job = list.jobs[jb];
        const int b = job.x, n = job.z, cta = list.first[jb];
        int h, half, row0, real;
        item_rows(a, job.y, rows, h, half, row0, real);
        if (r >= real) continue;
        const int gr = row0 + r;
        // place of piece i: the first or the second that its CTA left
        auto place = [&](int i) { return ((int64_t)(cta + i) * 2 + (i == 0 ? job.w : 0)) * rows + r; };
        // a piece without a finite score has seen nothing, or a NaN that its sum holds
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
        if (!wide) {
            const float2 ml = lane < n ? *reinterpret_cast<const float2*>(part_ml + place(lane) * 2) : make_float2(-INFINITY, 0.f);
            float4 o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                o[i] = i < n && col < a.cols ? *reinterpret_cast<const float4*>(part_o + place(i) * a.cols + col) : v;
            top = warp_max(ml.x);
            const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
            sum = warp_sum(ml.x == -INFINITY ? ml.y : ml.y * w);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float wi = __shfl_sync(0xffffffffu, w, i);
                v.x += o[i].x * wi;
                v.y += o[i].y * wi;
                v.z += o[i].z * wi;
                v.w += o[i].w * wi;
            }
        } else {
            __syncthreads();  // the unit before is done with shared memory
            for (int i = threadIdx.x; i < n; i += 128) {
                s_ml[i] = *reinterpret_cast<const float2*>(part_ml + place(i) * 2);
                top = fmaxf(top, s_ml[i].x);
            }
            top = warp_max(top);
            if (lane == 0) s_red[0][warp] = top;
            __syncthreads();
            top = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
            for (int i = threadIdx.x; i < n; i += 128) {
                const float m = s_ml[i].x, l = s_ml[i].y, w = m == -INFINITY ? 0.f : exp2f(m - top);
                s_ml[i].x = w;
                sum += m == -INFINITY ? l : l * w;
            }
            sum = warp_sum(sum);
            if (lane == 0) s_red[1][warp] = sum;
            __syncthreads();
            sum = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
            if (col < a.cols) {
#pragma unroll 8
                for (int i = warp; i < n; i += 4) {
                    const float4 o = *reinterpret_cast<const float4*>(part_o + place(i) * a.cols + col);
                    const float w = s_ml[i].x;
                    v.x += o.x * w;
                    v.y += o.y * w;
                    v.z += o.z * w;
                    v.w += o.w * w;
                }
            }
            s_o[threadIdx.x] = v;
            __syncthreads();
            if (warp == 0)
#pragma unroll
                for (int x = 1; x < 4; ++x) {
                    const float4 o = s_o[x * 32 + lane];
                    v.x += o.x;
                    v.y += o.y;
                    v.z += o.z;
                    v.w += o.w;
                }
        }
        if (col < a.cols && (!wide || warp == 0)) {
            const int j = gr / G, hq = h * G + gr - j * G;
            const int count = a.counts ? max(0, min(a.counts[b], a.S)) : a.S;
            const bool none = j >= count || sum == 0.f;
            const float inv = __fdividef(1.f, sum);
            uint2 res;
            res.x = none ? 0u : pack2<T>(v.x * inv, v.y * inv);
            res.y = none ? 0u : pack2<T>(v.z * inv, v.w * inv);
            *reinterpret_cast<uint2*>((T*)a.out + (((int64_t)b * a.S + j) * a.Hq + hq) * a.Dv + half * a.cols + col) = res;
        }
    }
}

// once per kernel and device
template <typename K>
static void allow_smem_once(K kernel, int bytes, std::atomic<uint64_t>& done) {
    const int dev = at::cuda::current_device();
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (done.load(std::memory_order_acquire) & bit) return;
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit, std::memory_order_release);
}

// Per CTA of the attention kernel: one join job and up to two pieces of `rows` rows.
struct Workspace {
    at::Tensor buf;
    int4* jobs;
    float *ml, *o;
    Workspace(const at::Tensor& like, int ctas, int rows, int Dv) {
        const int64_t n = (int64_t)ctas * 2 * rows;
        buf = at::empty({ctas * 4 + n * (Dv + 2)}, like.options().dtype(at::kFloat));
        jobs = reinterpret_cast<int4*>(buf.data_ptr());
        o = buf.data_ptr<float>() + ctas * 4;
        ml = o + n * Dv;
    }
};

// Launches a joining kernel (`per_sm` blocks an SM) that may be set up while the attention kernel before it runs.
template <typename... P, typename... X>
static void launch_behind(void (*kernel)(P...), int per_sm, cudaStream_t st, X... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(at::cuda::getCurrentDeviceProperties()->multiProcessorCount * per_sm));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
}
template <typename T>
static void launch_join(const AttnArgs& a, int rows, int ctas, const Workspace& ws, cudaStream_t st) {
    launch_behind(join_kernel<T>, 4, st, a, rows, ctas, (const int4*)ws.jobs, (const float*)ws.ml, (const float*)ws.o);
}

inline bool half_type(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

}  // namespace paged
}  // namespace atb
