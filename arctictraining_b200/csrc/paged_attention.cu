// SPDX-License-Identifier: Apache-2.0
// Attention of new tokens over the paged generation cache.
//
// Query j of a sequence stands at position p = starts + j and sees the cached positions max(0, p - window + 1) .. p:
// o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m), s_t = scale q.k_t, in one pass over the keys with the running maximum m.
// The latent form has one key row [latent | rotary] for all heads and the latent itself as value.
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
};

// ---- schedule ---------------------------------------------------------------------------------------------------------
// Work is counted in rounds of `NK` keys of one item (sequence, cache head, tile of query rows).  The rounds of all items
// stand in one line, each item's behind kLead empty ones that stand for what an item costs besides its keys (its queries,
// the pipeline's filling, the result: 2 to 3 us, a round 1.5 to 2 us), and every CTA takes an equal piece of the line, so a batch of very different lengths loads all SMs alike
// and a single long sequence is spread over all of them.  A CTA that covers an item alone writes the result; otherwise it
// leaves (maximum, sum, weighted values) of its piece in the workspace, and the join kernel adds the pieces in their
// order.  No atomics: the same inputs give the same bits.
constexpr int kLead = 2;
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
    r.rounds = kLead + max(1, (r.total - r.first + NK - 1) / NK);  // a sequence that sees nothing has one round, fully masked
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
__device__ __forceinline__ int4 join_job(const Pieces& pieces, int cta, int at, int to, int b, int line, const Range& rg) {
    if (cta == 0 || at >= to) return make_int4(0, 0, 0, 0);
    const int item = (at - line) / rg.rounds, s = line + item * rg.rounds;
    if (pieces.cta_of(s + kLead) != cta - 1) return make_int4(0, 0, 0, 0);
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

// ---- attention over grouped heads --------------------------------------------------------------------------------------
// Bound by memory: 4 Hq / Hkv flops a cached element.  A CTA of four warps serves the query rows (new token, head of the
// group) of one cache head, so that a cached row is read once for all of them; rows fill the 16-row side of the matrix
// instruction.  WR warps stand along the rows (1, 2 or 4 tiles of 16) and 4 / WR rings of warps along the keys: each ring
// streams its own keys through its own shared-memory stages (cp.async, kStages deep) and keeps its own running maximum,
// sum and weighted values; with one warp a ring nothing in the loop waits for another warp.  The rings are added at the end
// of a piece.  Eight-bit rows are turned into fp16 (exactly) on their way into the instruction, the scale of a key
// multiplies its score, and that of a value goes into the exponent of its probability, with a running maximum of its own,
// so that probabilities stay within (0, 1] whatever the scales are.
// Probabilities are rounded to the 16-bit type of the instruction (fp16 for e4m3 values): the same size of error as the
// final rounding of the result.  Scores, maxima, sums and weighted values are fp32.
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;

template <bool E4M3, int DP>
struct Shape {
    static constexpr int kRowBytes = DP * (E4M3 ? 1 : 2);
    // keys a warp loads per stage: 8 KB of keys and values where a row allows it
    static constexpr int kKeys = kRowBytes >= 256 ? 16 : kRowBytes == 128 ? 32 : 64;
    static constexpr int kRound = 4 * kKeys;  // keys of a round of the CTA
    // per warp and stage: keys, values, (scales)
    static constexpr int kStageBytes = 2 * kKeys * kRowBytes + (E4M3 ? 2 * kKeys * 4 : 0);
    static constexpr int kRingBytes = kStages * 4 * kStageBytes;
    static constexpr int kOutBytes = 4 * 16 * (DP + 4) * 4;  // the rings' results when they are added
    static constexpr int kSmem = kRingBytes > kOutBytes ? kRingBytes : kOutBytes;
};

template <typename T, bool E4M3, int DP, int WR>
__global__ void __launch_bounds__(128) rows_kernel(const AttnArgs a, int B, int4* __restrict__ jobs, float* __restrict__ part_ml,
                                                    float* __restrict__ part_o) {
    using Sh = Shape<E4M3, DP>;
    using P = typename std::conditional<E4M3, __half, T>::type;  // type of the matrix instruction
    constexpr int WK = 4 / WR, KW = Sh::kKeys, TK = KW * WR, NK = Sh::kRound, RB = Sh::kRowBytes;
    constexpr int CPR = RB / 16;         // 16-byte chunks of a row
    constexpr int KB = KW < 32 ? KW : 32;  // keys of one softmax step
    constexpr int kVal = E4M3 ? 8 : 4;     // registers of two 16-byte chunks of 16 values
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int scratch[10];
    __shared__ uint32_t s_valid[4][kStages][2];
    __shared__ float s_ml[4][16][2];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wr = warp % WR, wk = warp / WR;
    const int g = lane >> 2, c = lane & 3;
    const int G = a.Hq / a.Hkv, M = a.S * G;
    const int row_tiles = (M + 16 * WR - 1) / (16 * WR);
    const int per = a.Hkv * row_tiles;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the join kernel may be set up meanwhile
    int b, line, at, to;
    const Pieces pieces = find_piece<128>(a, B, NK, per, gridDim.x, blockIdx.x, at, to, b, line, scratch);
    Range rg;
    if (at < to) rg = seq_range(a, b, NK);
    if (threadIdx.x == 0) jobs[blockIdx.x] = join_job(pieces, blockIdx.x, at, to, b, line, rg);
    if (at >= to) return;
    const int began = at;

    const uint32_t ring = smem_addr(smem) + wk * WR * kStages * Sh::kStageBytes;
    // of a stage: keys of all warps of the ring, values, key scales, value scales
    constexpr int kK = 0, kV = WR * KW * RB, kSK = 2 * WR * KW * RB, kSV = kSK + WR * KW * 4, kStage = WR * Sh::kStageBytes;

    while (at < to) {
        while (at >= line + rg.rounds * per) {
            line += rg.rounds * per;
            ++b;
            rg = seq_range(a, b, NK);
        }
        const int item = (at - line) / rg.rounds;  // (cache head, row tile)
        const int v0 = at - line - item * rg.rounds, v1 = min(rg.rounds, v0 + (to - at));
        const int r0 = max(0, v0 - kLead), r1 = v1 - kLead;
        if (r1 <= r0) {  // only empty rounds of the item
            at += v1 - v0;
            continue;
        }
        const int h = item / row_tiles, row_base = (item - h * row_tiles) * 16 * WR + wr * 16;

        // query rows of this lane, and the positions that they see
        int row[2], hi[2], lo[2];
        uint32_t q[DP / 16][4];
        float fac[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            row[i] = row_base + g + 8 * i;
            const int j = min(row[i], M - 1) / G;
            hi[i] = (int)min((int64_t)rg.start + j, (int64_t)rg.total - 1);
            lo[i] = a.window > 0 ? (int)max((int64_t)0, (int64_t)rg.start + j + 1 - a.window) : 0;
            const T* src = (const T*)a.q + b * a.q_b + (int64_t)j * a.q_s + (int64_t)(h * G + min(row[i], M - 1) % G) * a.q_h;
            const bool real = row[i] < M;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                if (E4M3) {  // elements 4 c .. 4 c + 3 of the chunk, the order in which the keys' bytes arrive
                    uint2 u = make_uint2(0, 0);
                    if (real && k * 16 < a.D) u = *reinterpret_cast<const uint2*>(src + k * 16 + 4 * c);
                    q[k][i] = u.x;
                    q[k][i + 2] = u.y;
                } else {
                    const bool in = real && k * 16 < a.D;
                    q[k][i] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 2 * c) : 0u;
                    q[k][i + 2] = in ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8 + 2 * c) : 0u;
                }
            }
            // scores are multiplied by |scale| log2 e; a negative scale turns the queries' signs, and one of zero becomes tiny
            // so that a hidden key's -infinity stays what it is
            fac[i] = fmaxf(fabsf(a.scale), 1e-30f) * kLog2e;
            if (a.scale < 0.f) {
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    q[k][i] ^= 0x80008000u;
                    q[k][i + 2] ^= 0x80008000u;
                }
            }
        }
        if (E4M3 && std::is_same<T, bf16>::value) {
            // bf16 queries become fp16 after a power of two per row that brings their largest element to [2^14, 2^15):
            // exact down to 2^-28 of that element
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float m = 0.f;
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const float2 x = unpack2<T>(q[k][i]), y = unpack2<T>(q[k][i + 2]);
                    m = fmaxf(m, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
                }
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                const int e = (__float_as_uint(m) >> 23) & 255;
                const int field = e == 0 || e == 255 ? 127 : min(268 - e, 253);
                const float up = __uint_as_float((uint32_t)field << 23);
                fac[i] *= __uint_as_float((uint32_t)(254 - field) << 23);
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    const float2 x = unpack2<T>(q[k][i]), y = unpack2<T>(q[k][i + 2]);
                    q[k][i] = pack2<__half>(x.x * up, x.y * up);
                    q[k][i + 2] = pack2<__half>(y.x * up, y.y * up);
                }
            }
        }
        int min_hi = min(hi[0], hi[1]), max_lo = max(lo[0], lo[1]);
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            min_hi = min(min_hi, __shfl_xor_sync(0xffffffffu, min_hi, o));
            max_lo = max(max_lo, __shfl_xor_sync(0xffffffffu, max_lo, o));
        }

        const int key0 = rg.first + wk * TK;  // of the ring's tile in round 0 of the item
        const int n = r1 - r0;
        const int64_t head_rows = (int64_t)h * a.page;
        // Copies of one tile.  `even`: the keys that a warp loads lie in one page and rows are as wide as the stage's, so the
        // tile is one dense block; otherwise each lane looks up the page of its own key (64 keys: two) and the copies fetch
        // their row's place from it.  Positions advance by NK a tile: page and offset are carried along without a division.
        // The page id of the next tile is read a tile ahead.
        constexpr int LK = KW > 32 ? 2 : 1;
        const bool even = a.page % KW == 0 && a.D == DP;
        const int step_w = NK / a.page, step_off = NK - step_w * a.page;
        int look_key[LK], look_w[LK], look_off[LK], pid_next[LK];
#pragma unroll
        for (int x = 0; x < LK; ++x) {
            look_key[x] = key0 + r0 * NK + wr * KW + (even ? 0 : lane + 32 * x);
            look_w[x] = look_key[x] / a.page;
            look_off[x] = look_key[x] - look_w[x] * a.page;
        }
        const int* table = a.table + b * a.table_stride;
        auto look_up = [&](int t) {  // the page ids of tile t, whose positions look_* hold
#pragma unroll
            for (int x = 0; x < LK; ++x) {
                pid_next[x] = -1;
                const bool mine = even ? look_key[x] + KW > rg.low : (KW >= 32 || lane < KW) && look_key[x] >= rg.low;
                if (t < n && mine && look_key[x] < rg.total) pid_next[x] = table[look_w[x]];
            }
        };
        auto issue = [&](int t) {  // the copies of tile t of this piece; look_* and pid_next are its, and move on to the next
            if (t < n) {
                const int st = t % kStages;
                const uint32_t base = ring + st * kStage;
                constexpr int kIter = KW * CPR / 32;
                if (even) {
                    const int pid = pid_next[0], upto = rg.total - look_key[0], from = rg.low - look_key[0];
                    const bool ok = pid >= 0 && pid < a.P;
                    const int64_t r = head_rows + look_off[0];
                    const int64_t off = (ok ? pid * a.k_page + r * DP : 0) * (E4M3 ? 1 : 2) + lane * 16;
                    const uint8_t *ks = (const uint8_t*)a.k_pages + off, *vs = (const uint8_t*)a.v_pages + off;
                    // row i * 32 / CPR + lane / CPR: its chunk's place is exchanged within the row by the row's low bits
                    const int key = lane / CPR, ch = lane % CPR;
                    const uint32_t d = base + (wr * KW + key) * RB;
                    if (ok && upto >= KW && from <= 0) {
#pragma unroll
                        for (int i = 0; i < kIter; ++i) {
                            const uint32_t di = d + i * 512 + ((ch ^ key ^ (i * (32 / CPR) & 7)) & (CPR - 1)) * 16;
                            copy16(di + kK, ks + i * 512, true);
                            copy16(di + kV, vs + i * 512, true);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < kIter; ++i) {
                            const int k = i * (32 / CPR) + key;
                            const bool full = ok && k >= from && k < upto;
                            const uint32_t di = d + i * 512 + ((ch ^ key ^ (i * (32 / CPR) & 7)) & (CPR - 1)) * 16;
                            copy16(di + kK, full ? ks + i * 512 : a.k_pages, full);
                            copy16(di + kV, full ? vs + i * 512 : a.v_pages, full);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < LK; ++x) {
                        const int k = lane + 32 * x;
                        const bool full = ok && k >= from && k < upto;
                        if (E4M3 && k < KW) {
                            const int64_t so = full ? pid * a.ks_page + r + k : 0;
                            copy4(base + kSK + (wr * KW + k) * 4, a.k_scale + so, full);
                            copy4(base + kSV + (wr * KW + k) * 4, a.v_scale + so, full);
                        }
                        const uint32_t bits = __ballot_sync(0xffffffffu, full);
                        if (lane == 0) s_valid[warp][st][x] = bits;
                    }
                } else {
                    int64_t off[LK];
                    bool ok[LK];
#pragma unroll
                    for (int x = 0; x < LK; ++x) {
                        ok[x] = pid_next[x] >= 0 && pid_next[x] < a.P;
                        const int64_t r = head_rows + look_off[x];
                        off[x] = ok[x] ? pid_next[x] * a.k_page + r * a.D : 0;
                        const uint32_t bits = __ballot_sync(0xffffffffu, ok[x]);
                        if (lane == 0) s_valid[warp][st][x] = bits;
                        if (E4M3 && (KW >= 32 || lane < KW)) {
                            const int64_t so = ok[x] ? pid_next[x] * a.ks_page + r : 0;
                            const uint32_t d = base + kSK + (wr * KW + lane + 32 * x) * 4;
                            copy4(d, a.k_scale + so, ok[x]);
                            copy4(d + (kSV - kSK), a.v_scale + so, ok[x]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kIter; ++i) {
                        const int id = i * 32 + lane, key = id / CPR, ch = id % CPR;
                        const int64_t o = __shfl_sync(0xffffffffu, LK == 2 && i * 32 / CPR >= 32 ? off[LK - 1] : off[0], key & 31);
                        const bool full = __shfl_sync(0xffffffffu, LK == 2 && i * 32 / CPR >= 32 ? ok[LK - 1] : ok[0], key & 31) &&
                                          ch * 16 < a.D * (E4M3 ? 1 : 2);
                        const int64_t byte = full ? (E4M3 ? o : o * 2) + ch * 16 : 0;
                        const uint32_t d = base + (wr * KW + key) * RB + ((ch ^ (key & 7)) & (CPR - 1)) * 16;
                        copy16(d + kK, (const uint8_t*)a.k_pages + byte, full);
                        copy16(d + kV, (const uint8_t*)a.v_pages + byte, full);
                    }
                }
#pragma unroll
                for (int x = 0; x < LK; ++x) {
                    look_key[x] += NK;
                    look_w[x] += step_w;
                    look_off[x] += step_off;
                    if (look_off[x] >= a.page) {
                        look_off[x] -= a.page;
                        ++look_w[x];
                    }
                }
            }
            copies_commit();
        };
        auto ring_sync = [&]() {
            if (WR == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + wk), "n"(WR * 32) : "memory");
        };

        float o[DP / 8][4];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][x] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, mv[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

        look_up(0);
#pragma unroll
        for (int t = 0; t < kStages - 1; ++t) {
            issue(t);
            look_up(t + 1);
        }
        for (int t = 0; t < n; ++t) {
            copies_wait<kStages - 2>();
            ring_sync();
            issue(t + kStages - 1);
            look_up(t + kStages);
            const int st = t % kStages;
            const uint32_t base = ring + st * kStage;
            const int tile0 = key0 + (r0 + t) * NK;
#pragma unroll 1
            for (int kb = 0; kb < TK; kb += KB) {
                const int first = tile0 + kb;
                if (first >= rg.total) break;
                float s[KB / 8][4];
#pragma unroll
                for (int i = 0; i < KB / 8; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[i][x] = 0.f;
                // scores
#pragma unroll
                for (int kp = 0; kp < KB / 16; ++kp) {
                    const uint32_t krow = base + kK + (kb + kp * 16) * RB;
                    const int r = ((lane >> 4) << 3) + (lane & 7);
                    if (E4M3) {
#pragma unroll
                        for (int k = 0; k < DP / 16; k += 2) {
                            uint32_t f[4];
                            const int ch = (k + ((lane >> 3) & 1)) ^ (r & 7);
                            ldsm4(f, krow + r * RB + (ch & (CPR - 1)) * 16);
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                uint32_t b0, b1;
                                e4m3x4_to_f16x4(f[x], b0, b1);
                                mma<P>(s[2 * kp + (x >> 1)], q[k + (x & 1)], b0, b1);
                            }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k) {
                            uint32_t f[4];
                            const int ch = (2 * k + ((lane >> 3) & 1)) ^ (r & 7);
                            ldsm4(f, krow + r * RB + ch * 16);
                            mma<P>(s[2 * kp], q[k], f[0], f[1]);
                            mma<P>(s[2 * kp + 1], q[k], f[2], f[3]);
                        }
                    }
                }
                float lv[KB / 8][2];  // log2 of the values' scales
                if (E4M3) {
                    const float* sk = reinterpret_cast<const float*>(smem + (base - smem_addr(smem)) + kSK) + kb + 2 * c;
#pragma unroll
                    for (int i = 0; i < KB / 8; ++i) {
                        const float2 ks = *reinterpret_cast<const float2*>(sk + i * 8), sv = *reinterpret_cast<const float2*>(sk + WR * KW + i * 8);
                        lv[i][0] = __log2f(sv.x);
                        lv[i][1] = __log2f(sv.y);
#pragma unroll
                        for (int x = 0; x < 4; ++x) s[i][x] *= fac[x >> 1] * ((x & 1) ? ks.y : ks.x);
                    }
                }
                // mask, where a key of this step is hidden from some row
                const int wsrc = wk * WR + kb / KW;
                uint32_t valid = s_valid[wsrc][st][LK == 2 ? (kb % KW) / 32 : 0];
                const uint32_t all_bits = KB == 32 ? 0xffffffffu : 0xffffu;
                bool hidden = false;
                if (first + KB - 1 > min_hi || first < max_lo || (valid & all_bits) != all_bits) {
#pragma unroll
                    for (int i = 0; i < KB / 8; ++i)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            hidden = true;
                            const int k = i * 8 + 2 * c + (x & 1), pos = first + k;
                            if (pos > hi[x >> 1] || pos < lo[x >> 1] || !((valid >> k) & 1)) s[i][x] = -INFINITY;
                        }
                }
                // running maximum (of score + log2 value scale too), rescaling only when some row's grew
                float tm[2] = {-INFINITY, -INFINITY}, tv[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < KB / 8; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        tm[x >> 1] = fmaxf(tm[x >> 1], s[i][x]);
                        if (E4M3) tv[x >> 1] = fmaxf(tv[x >> 1], s[i][x] + lv[i][x & 1]);
                    }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    tm[i] = fmaxf(tm[i], __shfl_xor_sync(0xffffffffu, tm[i], 1));
                    tm[i] = fmaxf(tm[i], __shfl_xor_sync(0xffffffffu, tm[i], 2));
                    if (E4M3) {
                        tv[i] = fmaxf(tv[i], __shfl_xor_sync(0xffffffffu, tv[i], 1));
                        tv[i] = fmaxf(tv[i], __shfl_xor_sync(0xffffffffu, tv[i], 2));
                    } else {
                        tm[i] *= fac[i];
                        tv[i] = tm[i];
                    }
                }
                if (__any_sync(0xffffffffu, tm[0] > m[0] || tm[1] > m[1] || (E4M3 && (tv[0] > mv[0] || tv[1] > mv[1])))) {
                    float f[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float mn = fmaxf(m[i], tm[i]), vn = fmaxf(mv[i], tv[i]);
                        l[i] *= m[i] == -INFINITY ? 0.f : exp2f(m[i] - mn);
                        f[i] = mv[i] == -INFINITY ? 0.f : exp2f(mv[i] - vn);
                        m[i] = mn;
                        mv[i] = vn;
                    }
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[i][x] *= f[x >> 1];
                }
                const float mz[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
                const float vz[2] = {mv[0] == -INFINITY ? 0.f : mv[0], mv[1] == -INFINITY ? 0.f : mv[1]};
                uint32_t p[KB / 16][4];
#pragma unroll
                for (int i = 0; i < KB / 8; ++i) {
                    float e[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float pr = E4M3 ? exp2f(s[i][x] - mz[x >> 1]) : exp2f(fmaf(s[i][x], fac[x >> 1], -mz[x >> 1]));
                        l[x >> 1] += pr;
                        // a hidden key's scale may be anything
                        e[x] = !E4M3 ? pr : s[i][x] == -INFINITY ? 0.f : exp2f(s[i][x] + lv[i][x & 1] - vz[x >> 1]);
                    }
                    p[i / 2][(i & 1) * 2] = pack2<P>(e[0], e[1]);
                    p[i / 2][(i & 1) * 2 + 1] = pack2<P>(e[2], e[3]);
                }
                // weighted values
                auto load_values = [&](int kp, int k, uint32_t (&v)[kVal]) {
                    const uint32_t vrow = base + kV + (kb + kp * 16) * RB;
                    const int r = (((lane >> 3) & 1) << 3) + (lane & 7);
                    uint32_t f[4];
                    const int ch = (k + (lane >> 4)) ^ (r & 7);
                    ldsm4_t(f, vrow + r * RB + (ch & (CPR - 1)) * 16);
                    if constexpr (E4M3) {  // even and odd elements of a chunk become two tiles of eight columns
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            e4m3x4_to_f16x4(__byte_perm(f[x], 0, 0x3120), v[(x >> 1) * 4 + (x & 1)], v[(x >> 1) * 4 + 2 + (x & 1)]);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) v[x] = f[x];
                    }
                };
                if (hidden && M > G && values_not_finite<P, kVal, KB / 16, CPR>(load_values)) {
                    // A key that some rows see and others do not holds an infinity or a NaN: 0 times it is no 0.  Each token's
                    // rows get a product of their own in which the keys hidden from them are zeros.
                    const int last = min(row_base + 15, M - 1) / G;
                    for (int j = row_base / G; j <= last; ++j) {
                        const int hj = (int)min((int64_t)rg.start + j, (int64_t)rg.total - 1);
                        const int lj = a.window > 0 ? (int)max((int64_t)0, (int64_t)rg.start + j + 1 - a.window) : 0;
#pragma unroll 1
                        for (int kp = 0; kp < KB / 16; ++kp) {
                            uint32_t keep[2];
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int pos = first + kp * 16 + 8 * x + 2 * c;
                                keep[x] = (pos >= lj && pos <= hj ? 0xffffu : 0u) | (pos + 1 >= lj && pos + 1 <= hj ? 0xffff0000u : 0u);
                            }
#pragma unroll
                            for (int k = 0; k < CPR; k += 2) {
                                uint32_t v[kVal];
                                load_values(kp, k, v);
#pragma unroll
                                for (int x = 0; x < kVal / 2; ++x) {
                                    float add[4] = {0.f, 0.f, 0.f, 0.f};
                                    mma<P>(add, p[kp], v[2 * x] & keep[0], v[2 * x + 1] & keep[1]);
#pragma unroll
                                    for (int y = 0; y < 4; ++y)
                                        if (min(row[y >> 1], M - 1) / G == j) o[k * (kVal / 4) + x][y] += add[y];
                                }
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int kp = 0; kp < KB / 16; ++kp)
#pragma unroll
                        for (int k = 0; k < CPR; k += 2) {
                            uint32_t v[kVal];
                            load_values(kp, k, v);
#pragma unroll
                            for (int x = 0; x < kVal / 2; ++x) mma<P>(o[k * (kVal / 4) + x], p[kp], v[2 * x], v[2 * x + 1]);
                        }
                }
            }
        }
        copies_wait<0>();

        // add the rings: every warp leaves its 16 rows in shared memory (rows padded by 4 floats against bank conflicts)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        }
        __syncthreads();
        float* mine = reinterpret_cast<float*>(smem) + warp * 16 * (DP + 4);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // weighted values are in units of 2^mv: bring them to those of the sum, 2^m
            const float f = E4M3 ? (mv[i] == -INFINITY ? 0.f : exp2f(mv[i] - m[i])) : 1.f;
            float* dst = mine + (g + 8 * i) * (DP + 4);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                if (E4M3) {
                    *reinterpret_cast<float4*>(dst + k * 16 + 4 * c) =
                        make_float4(o[2 * k][2 * i] * f, o[2 * k + 1][2 * i] * f, o[2 * k][2 * i + 1] * f, o[2 * k + 1][2 * i + 1] * f);
                } else {
                    *reinterpret_cast<float2*>(dst + k * 16 + 2 * c) = make_float2(o[2 * k][2 * i], o[2 * k][2 * i + 1]);
                    *reinterpret_cast<float2*>(dst + k * 16 + 8 + 2 * c) = make_float2(o[2 * k + 1][2 * i], o[2 * k + 1][2 * i + 1]);
                }
            }
            if (c == 0) {
                s_ml[warp][g + 8 * i][0] = m[i];
                s_ml[warp][g + 8 * i][1] = l[i];
            }
        }
        __syncthreads();
        const bool whole = r0 == 0 && v1 == rg.rounds;
        const int slot = at == began ? 0 : 1;  // a CTA leaves at most two pieces: of the item it begins in and of the one it ends in
        const int64_t part = ((int64_t)blockIdx.x * 2 + slot) * 16 * WR;
        const int chunks = a.D / 8;
        const int tile_base = (item - h * row_tiles) * 16 * WR;
        const int count = a.counts ? max(0, min(a.counts[b], a.S)) : a.S;
        for (int u = threadIdx.x; u < 16 * WR * chunks; u += 128) {
            const int r = u / chunks, e = (u - r * chunks) * 8;
            const int rw = r / 16, rr = r % 16, gr = tile_base + r;
            if (gr >= M) continue;
            float top = -INFINITY, sum = 0.f, f[WK], v[8] = {};
#pragma unroll
            for (int k = 0; k < WK; ++k) top = fmaxf(top, s_ml[k * WR + rw][rr][0]);
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float mk = s_ml[k * WR + rw][rr][0];
                f[k] = mk == -INFINITY ? 0.f : exp2f(mk - top);
                // a ring without a finite score has seen nothing, or a NaN that its sum holds
                sum += mk == -INFINITY ? s_ml[k * WR + rw][rr][1] : f[k] * s_ml[k * WR + rw][rr][1];
                const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<float*>(smem) + ((k * WR + rw) * 16 + rr) * (DP + 4) + e);
                const float4 x = src[0], y = src[1];
                v[0] += f[k] * x.x; v[1] += f[k] * x.y; v[2] += f[k] * x.z; v[3] += f[k] * x.w;
                v[4] += f[k] * y.x; v[5] += f[k] * y.y; v[6] += f[k] * y.z; v[7] += f[k] * y.w;
            }
            if (whole) {
                const int j = gr / G, hq = h * G + gr - j * G;
                const float inv = j >= count || sum == 0.f ? 0.f : __fdividef(1.f, sum);
#pragma unroll
                for (int x = 0; x < 8; ++x) v[x] = j >= count || sum == 0.f ? 0.f : v[x] * inv;
                *reinterpret_cast<uint4*>((T*)a.out + (((int64_t)b * a.S + j) * a.Hq + hq) * a.D + e) = Vec8<T>::pack(v);
            } else {
                float4* dst = reinterpret_cast<float4*>(part_o + (part + r) * a.D + e);
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[1] = make_float4(v[4], v[5], v[6], v[7]);
                if (e == 0) {
                    part_ml[(part + r) * 2] = top;
                    part_ml[(part + r) * 2 + 1] = sum;
                }
            }
        }
        at += v1 - v0;
        __syncthreads();  // shared memory is refilled by the next piece
    }
}

// Adds the pieces of an item that several CTAs of the attention kernel worked on, in their order along the keys.  Such an item
// lies across the begin of some CTA's piece; the attention kernel left a job there.  Every block gathers the jobs, all in the
// same order, and the blocks share out (job, query row, 128 columns): a warp each where the items have few pieces, a block
// each, its warps taking pieces in turn, where some item has many.  The kernel is launched while the attention kernel runs, and
// waits for its end before it reads.  (Its pointers are not declared free of aliases: loads that are known to be invariant may
// be moved ahead of the wait.)
constexpr int kMaxCtas = 1024;
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const AttnArgs a, int rows, int ctas, const int4* jobs, const float* part_ml,
                                                   const float* part_o) {
    __shared__ int4 s_jobs[kMaxCtas];
    __shared__ int s_first[kMaxCtas], s_place[32], s_most;
    __shared__ float2 s_ml[kMaxCtas];
    __shared__ float s_red[2][4];
    __shared__ float4 s_o[128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = a.Hq / a.Hkv, M = a.S * G, row_tiles = (M + rows - 1) / rows;
    if (threadIdx.x == 0) s_most = 0;
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
        if (lane == 0) s_place[x * 4 + warp] = __popc(has[x]);
    }
    __syncthreads();
    int upto = s_place[lane];
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
            s_jobs[at] = mine[x];
            s_first[at] = threadIdx.x + 128 * x - 1;
            atomicMax(&s_most, mine[x].z);
        }
    }
    __syncthreads();
    const int used = row_tiles > 1 ? rows : M, slices = (a.Dv / 4 + 31) / 32;
    const int total = n_jobs * used * slices;
    const bool wide = s_most > 8;  // a block for each unit
    for (int u = wide ? blockIdx.x : blockIdx.x * 4 + warp; u < total; u += wide ? gridDim.x : gridDim.x * 4) {
        const int col = (u % slices) * 128 + lane * 4, rest = u / slices;
        const int r = rest % used, jb = rest / used;
        const int4 job = s_jobs[jb];
        const int b = job.x, n = job.z, cta = s_first[jb], h = job.y / row_tiles, gr = (job.y - h * row_tiles) * rows + r;
        if (gr >= M) continue;
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
                o[i] = i < n && col < a.Dv ? *reinterpret_cast<const float4*>(part_o + place(i) * a.Dv + col) : v;
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
            if (col < a.Dv) {
#pragma unroll 8
                for (int i = warp; i < n; i += 4) {
                    const float4 o = *reinterpret_cast<const float4*>(part_o + place(i) * a.Dv + col);
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
        if (col < a.Dv && (!wide || warp == 0)) {
            const int j = gr / G, hq = h * G + gr - j * G;
            const int count = a.counts ? max(0, min(a.counts[b], a.S)) : a.S;
            const bool none = j >= count || sum == 0.f;
            const float inv = __fdividef(1.f, sum);
            uint2 res;
            res.x = none ? 0u : pack2<T>(v.x * inv, v.y * inv);
            res.y = none ? 0u : pack2<T>(v.z * inv, v.w * inv);
            *reinterpret_cast<uint2*>((T*)a.out + (((int64_t)b * a.S + j) * a.Hq + hq) * a.Dv + col) = res;
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

template <typename T>
static void launch_join(const AttnArgs& a, int rows, int ctas, const Workspace& ws, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)at::cuda::getCurrentDeviceProperties()->multiProcessorCount * 4);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T>, a, rows, ctas, (const int4*)ws.jobs, (const float*)ws.ml, (const float*)ws.o));
}

template <typename T, bool E4M3, int DP, int WR>
static void launch_rows(const AttnArgs& a, int64_t B, const at::Tensor& q) {
    using Sh = Shape<E4M3, DP>;
    static std::atomic<uint64_t> done{0};
    allow_smem_once(rows_kernel<T, E4M3, DP, WR>, Sh::kSmem, done);
    const int rows = 16 * WR;
    const int ctas = std::min(kMaxCtas, at::cuda::getCurrentDeviceProperties()->multiProcessorCount * (Sh::kSmem > 110000 ? 1 : 2));
    const int G = a.Hq / a.Hkv;
    const int64_t row_tiles = ceil_div((int64_t)a.S * G, rows), items = a.Hkv * row_tiles;
    ATB_ARG(B * items * (ceil_div((int64_t)a.W * a.page, Sh::kRound) + 1 + kLead) < (int64_t(1) << 31),
            "paged_attention: too many sequences, query rows or positions for one call");
    const Workspace ws(q, ctas, rows, a.Dv);
    cudaStream_t st = current_stream();
    rows_kernel<T, E4M3, DP, WR><<<ctas, 128, Sh::kSmem, st>>>(a, (int)B, ws.jobs, ws.ml, ws.o);
    ATB_LAUNCH_CHECK();
    launch_join<T>(a, rows, ctas, ws, st);
}

template <typename T, bool E4M3, int DP>
static void launch_heads(const AttnArgs& a, int64_t B, const at::Tensor& q) {
    const int rows = a.S * (a.Hq / a.Hkv);
    if (rows <= 16) launch_rows<T, E4M3, DP, 1>(a, B, q);
    else if (rows <= 32) launch_rows<T, E4M3, DP, 2>(a, B, q);
    else launch_rows<T, E4M3, DP, 4>(a, B, q);
}

template <typename T, bool E4M3>
static void launch_dims(const AttnArgs& a, int64_t B, const at::Tensor& q) {
    if (a.D <= 64) launch_heads<T, E4M3, 64>(a, B, q);
    else if (a.D <= 128) launch_heads<T, E4M3, 128>(a, B, q);
    else launch_heads<T, E4M3, 256>(a, B, q);
}

// ---- latent attention --------------------------------------------------------------------------------------------------
// One key row [latent | rotary] for all heads, the latent being its value too: a row of 1152 bytes meets 2 x 16 MT query
// rows' products, so with 16 heads and one new token the memory still sets the pace.  A CTA of eight warps keeps the
// weighted values of its query rows in registers, 64 columns a warp, and takes 64 keys at a time.  Scores: the 36 depth
// steps of 16 are divided over four groups of warps (whose slice of the queries stays in registers) and the keys over two, so
// every key byte is read from shared memory once; the four partial sums meet in shared memory, where the softmax is taken by
// all threads.  Weighted values: every warp reads its own 64 columns of the same tile.  Precision is that of the grouped form.
constexpr int kLatent = 512, kRotary = 64, kJoint = kLatent + kRotary;

template <bool E4M3, int MT>
struct LatentShape {
    static constexpr int kKeys = 64;
    static constexpr int kRowBytes = kJoint * (E4M3 ? 1 : 2);
    static constexpr int kStageBytes = kKeys * kRowBytes + (E4M3 ? kKeys * 4 : 0);
    static constexpr int kRing = E4M3 ? 4 : 2;
    static constexpr int kScoreRow = 72;  // floats; 64 keys, spread over the banks
    static constexpr int kScores = kRing * kStageBytes;
    static constexpr int kProbs = kScores + 4 * 16 * MT * kScoreRow * 4;
    static_assert(4 * kScoreRow * 4 == kJoint * 2, "the queries pass through the scores' memory");
    static constexpr int kSmem = kProbs + 16 * MT * 128;
};

template <typename T, bool E4M3, int MT>
__global__ void __launch_bounds__(256) latent_kernel(const AttnArgs a, int B, int4* __restrict__ jobs, float* __restrict__ part_ml,
                                                    float* __restrict__ part_o) {
    using Sh = LatentShape<E4M3, MT>;
    using P = typename std::conditional<E4M3, __half, T>::type;
    constexpr int NK = Sh::kKeys, RB = Sh::kRowBytes, CPR = RB / 16, kRing = Sh::kRing, kRows = 16 * MT;
    constexpr int kSteps = 9;            // depth steps of a warp
    constexpr int kVal = E4M3 ? 8 : 4;   // registers of two 16-byte chunks of 16 values
    constexpr int kVChunks = 64 * (E4M3 ? 1 : 2) / 16;  // a warp's chunks of a value row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int scratch[10];
    __shared__ uint32_t s_valid[kRing][2];
    __shared__ float s_grow[kRows], s_fac[kRows], s_m[kRows], s_l[kRows];

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int dg = warp & 3, kh = warp >> 2;
    const int H = a.Hq, M = a.S * H, per = (M + kRows - 1) / kRows;

    int b, line, at, to;
    const Pieces pieces = find_piece<256>(a, B, NK, per, gridDim.x, blockIdx.x, at, to, b, line, scratch);
    Range rg;
    if (at < to) rg = seq_range(a, b, NK);
    if (threadIdx.x == 0) jobs[blockIdx.x] = join_job(pieces, blockIdx.x, at, to, b, line, rg);
    if (at >= to) return;
    const int began = at;
    const uint32_t ring = smem_addr(smem);
    float* scores = reinterpret_cast<float*>(smem + Sh::kScores);
    const uint32_t probs = smem_addr(smem) + Sh::kProbs;
    // place of a 16-byte chunk in a row: exchanged by the row's low bits so that eight rows meet different banks
    auto chunk_at = [](int key, int ch) { return (E4M3 ? ch ^ ((key >> 1) & 3) : ch ^ (key & 7)) * 16; };

    while (at < to) {
        while (at >= line + rg.rounds * per) {
            line += rg.rounds * per;
            ++b;
            rg = seq_range(a, b, NK);
        }
        const int item = (at - line) / rg.rounds;
        const int v0 = at - line - item * rg.rounds, v1 = min(rg.rounds, v0 + (to - at));
        const int r0 = max(0, v0 - kLead), r1 = v1 - kLead;
        if (r1 <= r0) {
            at += v1 - v0;
            continue;
        }
        const int n = r1 - r0, tile_base = item * kRows;
        const int* table = a.table + b * a.table_stride;

        // copies of tile t: four threads a key
        const int my_key = tid >> 2, my_part = tid & 3;
        int look_w, look_off, look_key = rg.first + r0 * NK + my_key, pid_next;
        look_w = look_key / a.page;
        look_off = look_key - look_w * a.page;
        const int step_w = NK / a.page, step_off = NK - step_w * a.page;
        auto look_up = [&](int t) {
            pid_next = -1;
            if (t < n && look_key < rg.total) pid_next = table[look_w];
        };
        auto issue = [&](int t) {
            if (t < n) {
                const int st = t % kRing;
                const uint32_t base = ring + st * Sh::kStageBytes + my_key * RB;
                const bool ok = pid_next >= 0 && pid_next < a.P;
                const uint8_t* src = (const uint8_t*)a.k_pages + (ok ? pid_next * a.k_page + (int64_t)look_off * a.D : 0) * (E4M3 ? 1 : 2);
                const int lat = a.D1 * (E4M3 ? 1 : 2), all = a.D * (E4M3 ? 1 : 2);
                constexpr int kLatChunks = kLatent * (E4M3 ? 1 : 2) / 16;
#pragma unroll
                for (int i = 0; i < CPR / 4; ++i) {
                    const int ch = i * 4 + my_part;
                    // narrower latents leave zeros between themselves and the rotary part
                    const int byte = ch < kLatChunks ? ch * 16 : lat + (ch - kLatChunks) * 16;
                    const bool full = ok && (ch < kLatChunks ? byte < lat : byte < all);
                    copy16(base + chunk_at(my_key, ch), full ? src + byte : (const uint8_t*)a.k_pages, full);
                }
                if (E4M3 && my_part == 0)
                    copy4(ring + st * Sh::kStageBytes + NK * RB + my_key * 4, a.k_scale + (ok ? pid_next * a.ks_page + look_off : 0), ok);
                // eight keys a warp: their bits, gathered from the first lane of each
                const uint32_t bits = __ballot_sync(0xffffffffu, ok);
                if (lane == 0) {
                    uint32_t eight = 0;
#pragma unroll
                    for (int k = 0; k < 8; ++k) eight |= ((bits >> (4 * k)) & 1u) << k;
                    reinterpret_cast<uint8_t*>(s_valid[st])[warp] = (uint8_t)eight;
                }
                look_key += NK;
                look_w += step_w;
                look_off += step_off;
                if (look_off >= a.page) {
                    look_off -= a.page;
                    ++look_w;
                }
            }
            copies_commit();
        };

        look_up(0);
#pragma unroll
        for (int t = 0; t < kRing - 1; ++t) {
            issue(t);
            look_up(t + 1);
        }

        // The queries pass through the score rows' memory (of the same size): joint rows [latent | rotary] with zeros where
        // there is no row or a width is narrower.
        {
            constexpr int kQChunks = kJoint / 8;
            for (int x = tid; x < kRows * kQChunks; x += 256) {
                const int r = x / kQChunks, ch = x - r * kQChunks, gr = tile_base + r, col = ch * 8;
                const int j = min(gr, M - 1) / H, h = min(gr, M - 1) - j * H;
                const T* src = col < kLatent ? (const T*)a.q + b * a.q_b + j * a.q_s + h * a.q_h + col
                                             : (const T*)a.q2 + b * a.q2_b + j * a.q2_s + h * a.q2_h + col - kLatent;
                const bool full = gr < M && (col < kLatent ? col < a.D1 : col - kLatent < a.D - a.D1);
                copy16(ring + Sh::kScores + r * (kJoint * 2) + ((ch ^ (r & 7)) * 16), full ? (const void*)src : a.q, full);
            }
            copies_commit();
            copies_wait<0>();
            __syncthreads();
        }
        const uint8_t* q_rows = smem + Sh::kScores;
        // bf16 queries against an 8-bit cache: the row's power of two (see the grouped form)
        if (E4M3 && std::is_same<T, bf16>::value) {
            for (int r = warp; r < kRows; r += 8) {
                float m = 0.f;
                for (int x = lane; x < kJoint / 2; x += 32) {
                    const float2 y = unpack2<T>(*reinterpret_cast<const uint32_t*>(q_rows + r * (kJoint * 2) + x * 4));
                    m = fmaxf(m, fmaxf(fabsf(y.x), fabsf(y.y)));
                }
                m = warp_max(m);
                const int e = (__float_as_uint(m) >> 23) & 255;
                if (lane == 0) s_fac[r] = __uint_as_float((uint32_t)(e == 0 || e == 255 ? 127 : min(268 - e, 253)) << 23);
            }
            __syncthreads();
        }
        // this warp's depth slice of them
        uint32_t q[MT][kSteps][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = mt * 16 + g + 8 * i;
                const uint8_t* row = q_rows + r * (kJoint * 2);
                const float up = E4M3 && std::is_same<T, bf16>::value ? s_fac[r] : 1.f;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    const int ch = (dg * kSteps + k) * 2;
                    uint32_t x, y;
                    if (E4M3) {  // elements 4 c .. 4 c + 3, the order in which the keys' bytes arrive
                        const uint2 u = *reinterpret_cast<const uint2*>(row + (((ch + (c >> 1)) ^ (r & 7)) * 16) + (c & 1) * 8);
                        x = u.x;
                        y = u.y;
                    } else {
                        x = *reinterpret_cast<const uint32_t*>(row + ((ch ^ (r & 7)) * 16) + c * 4);
                        y = *reinterpret_cast<const uint32_t*>(row + (((ch + 1) ^ (r & 7)) * 16) + c * 4);
                    }
                    if (a.scale < 0.f) {
                        x ^= 0x80008000u;
                        y ^= 0x80008000u;
                    }
                    if (E4M3 && std::is_same<T, bf16>::value) {
                        const float2 fx = unpack2<T>(x), fy = unpack2<T>(y);
                        x = pack2<__half>(fx.x * up, fx.y * up);
                        y = pack2<__half>(fy.x * up, fy.y * up);
                    }
                    q[mt][k][i] = x;
                    q[mt][k][i + 2] = y;
                }
            }

        // softmax: kLanes threads a row, kCols keys each
        constexpr int kLanes = 256 / kRows, kCols = NK / kLanes;
        const int srow = tid / kLanes, scol = (tid % kLanes) * kCols;
        const int sj = min(tile_base + srow, M - 1) / H;
        const int hi = (int)min((int64_t)rg.start + sj, (int64_t)rg.total - 1);
        float fac = fmaxf(fabsf(a.scale), 1e-30f) * kLog2e;
        if (E4M3 && std::is_same<T, bf16>::value) fac *= __uint_as_float((254u << 23) - __float_as_uint(s_fac[srow]));
        float m = -INFINITY, mv = -INFINITY, l = 0.f;
        float o[MT][8][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[mt][i][x] = 0.f;

        for (int t = 0; t < n; ++t) {
            copies_wait<kRing - 2>();
            __syncthreads();  // tile t is here; every warp is done with tile t - 1
            issue(t + kRing - 1);
            look_up(t + kRing);
            const int st = t % kRing;
            const uint32_t base = ring + st * Sh::kStageBytes;
            const int first = rg.first + (r0 + t) * NK;
            // scores of this warp's 32 keys and depth slice
            {
                float s[MT][4][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int x = 0; x < 4; ++x) s[mt][i][x] = 0.f;
                const int r = ((lane >> 4) << 3) + (lane & 7), half = (lane >> 3) & 1;
#pragma unroll
                for (int kp = 0; kp < 2; ++kp) {
                    const int key = kh * 32 + kp * 16 + r;
                    const uint32_t krow = base + key * RB;
                    if (E4M3) {
#pragma unroll
                        for (int k = 0; k < kSteps; k += 2) {
                            uint32_t f[4];
                            // the ninth step has no partner: its second half is read again and not used
                            const int ch = dg * kSteps + min(k + half, kSteps - 1);
                            ldsm4(f, krow + chunk_at(key, ch));
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                if (k + (x & 1) >= kSteps) continue;
                                uint32_t b0, b1;
                                e4m3x4_to_f16x4(f[x], b0, b1);
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) mma<P>(s[mt][2 * kp + (x >> 1)], q[mt][k + (x & 1)], b0, b1);
                            }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            uint32_t f[4];
                            ldsm4(f, krow + chunk_at(key, 2 * (dg * kSteps + k) + half));
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                mma<P>(s[mt][2 * kp], q[mt][k], f[0], f[1]);
                                mma<P>(s[mt][2 * kp + 1], q[mt][k], f[2], f[3]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float* dst = scores + (dg * kRows + mt * 16 + g) * Sh::kScoreRow + kh * 32 + i * 8 + 2 * c;
                        *reinterpret_cast<float2*>(dst) = make_float2(s[mt][i][0], s[mt][i][1]);
                        *reinterpret_cast<float2*>(dst + 8 * Sh::kScoreRow) = make_float2(s[mt][i][2], s[mt][i][3]);
                    }
            }
            __syncthreads();
            // softmax of the tile
            {
                float x[kCols], lv[kCols];
#pragma unroll
                for (int i = 0; i < kCols; i += 4) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const float4 y = *reinterpret_cast<const float4*>(scores + (d * kRows + srow) * Sh::kScoreRow + scol + i);
                        v.x += y.x;
                        v.y += y.y;
                        v.z += y.z;
                        v.w += y.w;
                    }
                    x[i] = v.x * fac;
                    x[i + 1] = v.y * fac;
                    x[i + 2] = v.z * fac;
                    x[i + 3] = v.w * fac;
                }
                if (E4M3) {
                    const float* sc = reinterpret_cast<const float*>(smem + st * Sh::kStageBytes + NK * RB) + scol;
#pragma unroll
                    for (int i = 0; i < kCols; ++i) {
                        const float y = sc[i];
                        x[i] *= y;
                        lv[i] = __log2f(y);
                    }
                }
                const uint32_t valid = s_valid[st][scol >> 5] >> (scol & 31);
                float tm = -INFINITY, tv = -INFINITY;
#pragma unroll
                for (int i = 0; i < kCols; ++i) {
                    if (first + scol + i > hi || !((valid >> i) & 1)) x[i] = -INFINITY;
                    tm = fmaxf(tm, x[i]);
                    if (E4M3) tv = fmaxf(tv, x[i] + lv[i]);
                }
#pragma unroll
                for (int d = 1; d < kLanes; d <<= 1) {
                    tm = fmaxf(tm, __shfl_xor_sync(0xffffffffu, tm, d));
                    if (E4M3) tv = fmaxf(tv, __shfl_xor_sync(0xffffffffu, tv, d));
                }
                if (!E4M3) tv = tm;
                const float mn = fmaxf(m, tm), vn = fmaxf(mv, tv);
                l *= m == -INFINITY ? 0.f : exp2f(m - mn);
                if (tid % kLanes == 0) s_grow[srow] = mv == -INFINITY ? 0.f : exp2f(mv - vn);
                m = mn;
                mv = vn;
                const float mz = m == -INFINITY ? 0.f : m, vz = mv == -INFINITY ? 0.f : mv;
                uint32_t w[kCols / 2];
#pragma unroll
                for (int i = 0; i < kCols; i += 2) {
                    float e[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float pr = exp2f(x[i + k] - mz);
                        l += pr;
                        e[k] = !E4M3 ? pr : x[i + k] == -INFINITY ? 0.f : exp2f(x[i + k] + lv[i + k] - vz);
                    }
                    w[i / 2] = pack2<P>(e[0], e[1]);
                }
                uint8_t* dst = smem + Sh::kProbs + srow * 128;
                const int ch = scol / 8;
                if (kCols == 4) *reinterpret_cast<uint2*>(dst + ((ch ^ (srow & 7)) * 16) + (scol & 4) * 2) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint4*>(dst + ((ch ^ (srow & 7)) * 16)) = make_uint4(w[0], w[1], w[kCols / 2 - 2], w[kCols / 2 - 1]);
            }
            __syncthreads();
            // weighted values of this warp's 64 columns
            {
                bool grew = false;
                float f[MT][2];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        f[mt][i] = s_grow[mt * 16 + g + 8 * i];
                        grew = grew || f[mt][i] != 1.f;
                    }
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[mt][i][x] *= f[mt][x >> 1];
                }
                auto load_probs = [&](int mt, int kp, uint32_t (&p)[4]) {
                    const int r = mt * 16 + (lane & 15);
                    ldsm4(p, probs + r * 128 + (((kp * 2 + (lane >> 4)) ^ (r & 7)) * 16));
                };
                auto load_values = [&](int kp, int k, uint32_t (&v)[kVal]) {
                    const int key = kp * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
                    uint32_t x[4];
                    ldsm4_t(x, base + key * RB + chunk_at(key, warp * kVChunks + k + (lane >> 4)));
                    if constexpr (E4M3) {
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            e4m3x4_to_f16x4(__byte_perm(x[y], 0, 0x3120), v[(y >> 1) * 4 + (y & 1)], v[(y >> 1) * 4 + 2 + (y & 1)]);
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; ++y) v[y] = x[y];
                    }
                };
                const bool hidden = a.S > 1 && first + NK - 1 > rg.start;
                if (hidden && values_not_finite<P, kVal, 4, kVChunks>(load_values)) {
                    // see the grouped form: each new token's rows get a product without the keys hidden from them
                    const int last = min(tile_base + kRows - 1, M - 1) / H;
                    for (int j = tile_base / H; j <= last; ++j) {
                        const int hj = (int)min((int64_t)rg.start + j, (int64_t)rg.total - 1);
#pragma unroll 1
                        for (int kp = 0; kp < 4; ++kp) {
                            uint32_t keep[2], p[MT][4];
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int pos = first + kp * 16 + 8 * x + 2 * c;
                                keep[x] = (pos <= hj ? 0xffffu : 0u) | (pos + 1 <= hj ? 0xffff0000u : 0u);
                            }
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) load_probs(mt, kp, p[mt]);
#pragma unroll
                            for (int k = 0; k < kVChunks; k += 2) {
                                uint32_t v[kVal];
                                load_values(kp, k, v);
#pragma unroll
                                for (int x = 0; x < kVal / 2; ++x)
#pragma unroll
                                    for (int mt = 0; mt < MT; ++mt) {
                                        float add[4] = {0.f, 0.f, 0.f, 0.f};
                                        mma<P>(add, p[mt], v[2 * x] & keep[0], v[2 * x + 1] & keep[1]);
#pragma unroll
                                        for (int y = 0; y < 4; ++y)
                                            if (min(tile_base + mt * 16 + g + 8 * (y >> 1), M - 1) / H == j) o[mt][k * (kVal / 4) + x][y] += add[y];
                                    }
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int kp = 0; kp < 4; ++kp) {
                        uint32_t p[MT][4];
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) load_probs(mt, kp, p[mt]);
#pragma unroll
                        for (int k = 0; k < kVChunks; k += 2) {
                            uint32_t v[kVal];
                            load_values(kp, k, v);
#pragma unroll
                            for (int x = 0; x < kVal / 2; ++x)
#pragma unroll
                                for (int mt = 0; mt < MT; ++mt) mma<P>(o[mt][k * (kVal / 4) + x], p[mt], v[2 * x], v[2 * x + 1]);
                        }
                    }
                }
            }
        }
        copies_wait<0>();
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        __syncthreads();  // the last tile's s_grow has been read
        if (tid % kLanes == 0) {
            s_m[srow] = m;
            s_l[srow] = l;
            s_grow[srow] = !E4M3 ? 1.f : mv == -INFINITY ? 0.f : exp2f(mv - m);  // weighted values are in units of 2^mv
        }
        __syncthreads();
        const bool whole = r0 == 0 && v1 == rg.rounds;
        const int slot = at == began ? 0 : 1;
        const int64_t part = ((int64_t)blockIdx.x * 2 + slot) * kRows;
        const int count = a.counts ? max(0, min(a.counts[b], a.S)) : a.S;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = mt * 16 + g + 8 * i, gr = tile_base + r;
                if (gr >= M) continue;
                const float f = s_grow[r], sum = s_l[r];
                const bool none = gr / H >= count || sum == 0.f;
                const float inv = whole ? __fdividef(f, sum) : f;
                T* out = (T*)a.out + (((int64_t)b * a.S * H) + gr) * a.Dv;
                float* dst = part_o + (part + r) * a.Dv;
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // 16 columns: two tiles of eight, or (8-bit) of even and of odd columns
                    const int col = warp * 64 + k * 16;
                    if (col >= a.Dv) continue;
                    float e[4] = {o[mt][2 * k][2 * i] * inv, o[mt][2 * k][2 * i + 1] * inv, o[mt][2 * k + 1][2 * i] * inv,
                                  o[mt][2 * k + 1][2 * i + 1] * inv};
                    const int at0 = E4M3 ? col + 4 * c : col + 2 * c, at1 = E4M3 ? at0 + 2 : at0 + 8;
                    if (E4M3) {
                        const float x = e[1];
                        e[1] = e[2];
                        e[2] = x;
                    }
                    if (whole) {
                        *reinterpret_cast<uint32_t*>(out + at0) = none ? 0u : pack2<T>(e[0], e[1]);
                        *reinterpret_cast<uint32_t*>(out + at1) = none ? 0u : pack2<T>(e[2], e[3]);
                    } else {
                        *reinterpret_cast<float2*>(dst + at0) = make_float2(e[0], e[1]);
                        *reinterpret_cast<float2*>(dst + at1) = make_float2(e[2], e[3]);
                    }
                }
                if (!whole && warp == 0 && c == 0) {
                    part_ml[(part + r) * 2] = s_m[r];
                    part_ml[(part + r) * 2 + 1] = sum;
                }
            }
        at += v1 - v0;
        __syncthreads();
    }
}

template <typename T, bool E4M3, int MT>
static void launch_latent_rows(const AttnArgs& a, int64_t B, const at::Tensor& q) {
    using Sh = LatentShape<E4M3, MT>;
    static std::atomic<uint64_t> done{0};
    allow_smem_once(latent_kernel<T, E4M3, MT>, Sh::kSmem, done);
    const int rows = 16 * MT, ctas = std::min(kMaxCtas, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
    const int64_t items = ceil_div((int64_t)a.S * a.Hq, rows);
    ATB_ARG(B * items * (ceil_div((int64_t)a.W * a.page, Sh::kKeys) + 1 + kLead) < (int64_t(1) << 31),
            "paged_latent_attention: too many sequences, query rows or positions for one call");
    const Workspace ws(q, ctas, rows, a.Dv);
    cudaStream_t st = current_stream();
    latent_kernel<T, E4M3, MT><<<ctas, 256, Sh::kSmem, st>>>(a, (int)B, ws.jobs, ws.ml, ws.o);
    ATB_LAUNCH_CHECK();
    launch_join<T>(a, rows, ctas, ws, st);
}

template <typename T, bool E4M3>
static void launch_latent(const AttnArgs& a, int64_t B, const at::Tensor& q) {
    if (a.S * a.Hq <= 16) launch_latent_rows<T, E4M3, 1>(a, B, q);
    else launch_latent_rows<T, E4M3, 2>(a, B, q);
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
    ATB_ARG(k_pages.stride(0) == v_pages.stride(0) && (!k_scale.has_value() || k_scale->stride(0) == v_scale->stride(0)), op,
            ": the pages of keys and values must lie equally far apart");
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
    if (k_pages.size(0) == 0 || table.size(1) == 0) return out.zero_();
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
    const bool f8 = is_e4m3(k_pages);
    if (q.scalar_type() == at::kBFloat16) f8 ? launch_dims<bf16, true>(a, B, q) : launch_dims<bf16, false>(a, B, q);
    else f8 ? launch_dims<__half, true>(a, B, q) : launch_dims<__half, false>(a, B, q);
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
    if (pages.size(0) == 0 || table.size(1) == 0) return out.zero_();
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
    const bool f8 = is_e4m3(pages);
    if (q.scalar_type() == at::kBFloat16) f8 ? launch_latent<bf16, true>(a, B, q) : launch_latent<bf16, false>(a, B, q);
    else f8 ? launch_latent<__half, true>(a, B, q) : launch_latent<__half, false>(a, B, q);
    return out;
}

}  // namespace atb
