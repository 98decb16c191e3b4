// SPDX-License-Identifier: Apache-2.0
// Attention of new tokens over the paged generation cache, heads in groups.
#include "paged_attention.cuh"

namespace atb {
namespace paged {

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
// Measured: four 8-bit caches of up to 131000 positions (807 MB) 138 us, 91 % of a plain copy's rate, in a short replay at 1965 MHz;
// 162 us, 77 %, after a second of such calls, when the power limit lowers the clocks.  64 sequences of 17 to 6100 positions (402 MB)
// 73 us, 85 %, and over 8-bit rows (208 MB) 54 us, 59 %; 256-wide heads, 24 sequences of 4000 positions (787 MB) 136 us, 89 %; one
// sequence of 777 positions 10.6 us (two launches and four dependent loads: lengths, page, keys, pieces).  Drafts of five tokens in
// fp16 layers of 64-wide heads with a window of 4096 (156 MB) 44 us, 55 %: eight warps an SM, stalled on fixed latencies.  Many new
// tokens are far from the floor (8 sequences of 4000 positions, 32 heads on 8: 64 tokens 180 us of 22, 128 tokens 365 us of 41):
// every tile of 64 query rows reads all keys of its cache head, those hidden from all its rows too.
constexpr int kStages = 3;

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
    if (threadIdx.x == 0) jobs[blockIdx.x] = join_job(a, pieces, blockIdx.x, at, to, b, line, rg);
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
        const int r0 = max(0, v0 - a.lead), r1 = v1 - a.lead;
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
            lo[i] = a.window > 0 ? (int)min((int64_t)rg.total, max((int64_t)0, (int64_t)rg.start + j + 1 - a.window)) : 0;
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
                        const int lj = a.window > 0 ? (int)min((int64_t)rg.total, max((int64_t)0, (int64_t)rg.start + j + 1 - a.window)) : 0;
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

template <typename T, bool E4M3, int DP, int WR>
static void launch_rows(AttnArgs a, int64_t B, const at::Tensor& q) {
    using Sh = Shape<E4M3, DP>;
    static std::atomic<uint64_t> done{0};
    allow_smem_once(rows_kernel<T, E4M3, DP, WR>, Sh::kSmem, done);
    const int rows = 16 * WR;
    const int ctas = std::min(kMaxCtas, at::cuda::getCurrentDeviceProperties()->multiProcessorCount * (Sh::kSmem > 110000 ? 1 : 2));
    const int G = a.Hq / a.Hkv;
    const int64_t row_tiles = ceil_div((int64_t)a.S * G, rows), items = a.Hkv * row_tiles;
    ATB_ARG(B * items * (ceil_div((int64_t)a.W * a.page, Sh::kRound) + 3) < (int64_t(1) << 31),
            "paged_attention: too many sequences, query rows or positions for one call");
    a.cols = a.Dv;
    a.halves = 1;
    a.token_tiles = 0;
    a.lead = 2;
    const Workspace ws(q, ctas, rows, a.cols);
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

}  // namespace atb
