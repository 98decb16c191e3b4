// SPDX-License-Identifier: Apache-2.0
// Attention of new tokens over the paged latent cache (absorbed multi-head latent attention).
#include "paged_attention.cuh"
#include "ptx_sm100.cuh"

namespace atb {

CUtensorMap make_tmap_bf16_public(const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows);
at::Tensor& gemm_error_flag(const at::Device& dev);

namespace paged {

// ---- latent attention --------------------------------------------------------------------------------------------------
// One key row [latent | rotary] for all heads, the latent being its value too: a row of 1152 bytes meets 2 x 16 MT query
// rows' products, so with 16 heads and one new token the memory still sets the pace.  A CTA of eight warps keeps the
// weighted values of its query rows in registers, 64 columns a warp, and takes 64 keys at a time.  Scores: the 36 depth
// steps of 16 are divided over four groups of warps (whose slice of the queries stays in registers) and the keys over two, so
// every key byte is read from shared memory once; the four partial sums meet in shared memory, where the softmax is taken by
// all threads.  Weighted values: every warp reads its own 64 columns of the same tile.  Precision is that of the grouped form.
// Measured with 16 heads: one sequence of 4003 positions 15 us; 89585 positions in 32 sequences (104 MB) 34 us, 47 % of a plain
// copy's rate (a tile of 64 keys takes 2 us, 1.75 of them its 74 KB; ten tiles a CTA do not hide the 7 us of an item's begin and
// end and the joining), 8-bit rows (53 MB) 33 us, 25 %; 32 heads 47 and 49 us.
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
    if (threadIdx.x == 0) jobs[blockIdx.x] = join_job(a, pieces, blockIdx.x, at, to, b, line, rg);
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
        const int r0 = max(0, v0 - a.lead), r1 = v1 - a.lead;
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
static void launch_latent_rows(AttnArgs a, int64_t B, const at::Tensor& q) {
    using Sh = LatentShape<E4M3, MT>;
    static std::atomic<uint64_t> done{0};
    allow_smem_once(latent_kernel<T, E4M3, MT>, Sh::kSmem, done);
    const int rows = 16 * MT, ctas = std::min(kMaxCtas, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
    const int64_t items = ceil_div((int64_t)a.S * a.Hq, rows);
    ATB_ARG(B * items * (ceil_div((int64_t)a.W * a.page, Sh::kKeys) + 3) < (int64_t(1) << 31),
            "paged_latent_attention: too many sequences, query rows or positions for one call");
    a.cols = a.Dv;
    a.halves = 1;
    a.token_tiles = 0;
    a.lead = 2;
    const Workspace ws(q, ctas, rows, a.cols);
    cudaStream_t st = current_stream();
    latent_kernel<T, E4M3, MT><<<ctas, 256, Sh::kSmem, st>>>(a, (int)B, ws.jobs, ws.ml, ws.o);
    ATB_LAUNCH_CHECK();
    launch_join<T>(a, rows, ctas, ws, st);
}

// ---- latent attention of many heads -------------------------------------------------------------------------------------
// Many heads of a token (the form is taken from 33 on) fill the 128 rows of the tensor core's accumulator, and 242 flops a cached
// byte (128 heads) make the matrix rate the bound.  One CTA takes the 128 rows of a token's heads and half of the 512 value
// columns: weighted values 256, two score buffers of 32 keys, and 384 of the 576 query columns as left operand fill the 512
// columns of tensor memory; the other 192 query columns and four stages of 32 keys lie in shared memory.  A left operand in
// tensor memory is not read again from shared memory for each of the 36 depth steps, whose bandwidth bounds a product with
// only 32 columns.  The price of halves is that both compute the scores: 1.5 times the multiply-adds of one CTA per row tile,
// whose 512 value columns alone would fill tensor memory.
// Warps 0-3: a query row a thread: scores out of tensor memory, softmax, probabilities back in their place.  Warps 4-7 fetch keys
// (8-bit ones are turned into fp16 on the way).  Warp 8 issues the products; scores of the next tile run ahead of the values
// of this one.  All keys that a row tile sees are the same for its rows (one token), so hidden keys are never fetched.
// The accumulator is rescaled only when a row's maximum grew by more than 2^8.  All waits are bounded.
// Measured: 128 heads, 89585 positions in 32 sequences (25 GFLOP, 112 MB) 60 us: the products take 24 of them (1070 cycles a
// tile of 32 keys, as the instruction rates say), queries, first keys, results and the joining of a CTA's two or three pieces
// the rest, one after the other; 8-bit 79 us (the softmax, and the pass for the queries' magnitudes); one sequence of 60000 positions
// 46 us; 4 sequences of 4000 positions with 64 new tokens 384 us of 172.
namespace tc {
constexpr int kThreads = 288, kKeys = 32, kRing = 4, kRows = 128, kCols = 256;
constexpr int kSub = kKeys * 128;                       // 64 columns of a stage, 128-byte swizzled rows
constexpr int kStage = kJoint / 64 * kSub;
constexpr int kQTmem = 384, kQSub = kRows * 128;        // query columns in tensor memory; 64 columns of the others
constexpr int kQ = 0, kK = (kJoint - kQTmem) / 64 * kQSub, kScale = kK + kRing * kStage, kValid = kScale + 2 * kRing * kKeys * 4;
constexpr int kBars = kValid + kRing * 4 + 8, kSmem0 = kBars + 32 * 8 + 64;
constexpr int kSpare = (kSmem0 + 1023) / 1024 * 1024, kSmem = kSpare + 2 * kQSub;  // two more buffers of 64 query columns
static_assert(kBars % 8 == 0 && kK % 1024 == 0 && kQTmem == 6 * 64 && kJoint == 9 * 64, "aligned, and parts as the queries are fetched");
constexpr uint32_t kS = 256, kQCol = 320;               // columns of tensor memory: values 0, scores 256 and 288, queries 320
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr float kGrow = 8.f;

// What a role has issued must not outlive the CTA, also where another role gave up: waits for it (bounded), whatever the others do.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity) {
    const uint64_t t0 = ptx::globaltimer_ns();
    while (!ptx::mbar_try_wait(bar, parity))
        if (ptx::globaltimer_ns() - t0 > 100000000ull) return;
}

struct Piece {
    int b, item, r0, n, row0, rows, half, token;
    bool whole, first;
    Range rg;
};
// The pieces of one CTA in their order: every role walks the same ones.
struct Walk {
    int at, to, began, b, line, per;
    Range rg;
    __device__ __forceinline__ bool next(const AttnArgs& a, Piece& p) {
        while (at < to) {
            while (at >= line + rg.rounds * per) {
                line += rg.rounds * per;
                ++b;
                rg = seq_range(a, b, kKeys);
            }
            p.item = (at - line) / rg.rounds;
            const int v0 = at - line - p.item * rg.rounds, v1 = min(rg.rounds, v0 + (to - at));
            p.first = at == began;
            at += v1 - v0;
            p.r0 = max(0, v0 - a.lead);
            p.n = v1 - a.lead - p.r0;
            if (p.n <= 0) continue;
            p.b = b;
            p.rg = rg;
            p.whole = p.r0 == 0 && v1 == rg.rounds;
            int h;
            item_rows(a, p.item, kRows, h, p.half, p.row0, p.rows);
            p.token = p.row0 / a.Hq;
            return true;
        }
        return false;
    }
};

template <typename Q, bool E4M3>
__global__ void __launch_bounds__(kThreads, 1)
latent_tc_kernel(const __grid_constant__ CUtensorMap tmap, int page_rows, const AttnArgs a, int B, int4* __restrict__ jobs,
                 float* __restrict__ part_ml, float* __restrict__ part_o, int* error_flag) {
    using P = typename std::conditional<E4M3, __half, Q>::type;
    extern __shared__ __align__(1024) uint8_t smem[];
    int* scratch = reinterpret_cast<int*>(smem + kBars + 32 * 8);  // no static memory: the tiles' alignment
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kBars);
    uint64_t *k_full = bars, *k_empty = bars + kRing, *s_full = bars + 2 * kRing, *p_full = s_full + 2, *pv_done = p_full + 2,
             *q_full = pv_done + 2, *q_sync = q_full + 1, *drained = q_sync + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 24);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* s_scale = reinterpret_cast<float*>(smem + kScale);
    uint32_t* s_valid = reinterpret_cast<uint32_t*>(smem + kValid);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    Walk walk;
    walk.per = a.S * a.token_tiles * a.halves;
    const Pieces pieces = find_piece<kThreads>(a, B, kKeys, walk.per, gridDim.x, blockIdx.x, walk.at, walk.to, walk.b, walk.line, scratch);
    if (walk.at < walk.to) walk.rg = seq_range(a, walk.b, kKeys);
    if (threadIdx.x == 0) jobs[blockIdx.x] = join_job(a, pieces, blockIdx.x, walk.at, walk.to, walk.b, walk.line, walk.rg);
    if (walk.at >= walk.to) return;
    walk.began = walk.at;
    if ((ptx::smem_u32(smem) & 1023u) != 0) {  // the swizzled tiles need 1024-byte alignment
        if (threadIdx.x == 0) atomicCAS(error_flag, 0, (0x30 << 8) | 1);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            ptx::mbar_init(&k_full[i], 128);
            ptx::mbar_init(&k_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ptx::mbar_init(&s_full[i], 1);
            ptx::mbar_init(&p_full[i], 128);
            ptx::mbar_init(&pv_done[i], 1);
        }
        ptx::mbar_init(q_full, 128);
        ptx::mbar_init(q_sync, 128);
        ptx::mbar_init(drained, 1);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
    }
    if (warp == 8) {
        ptx::tmem_alloc(tmem_slot, 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    Piece p;

    if (warp >= 4 && warp < 8) {
        // -------------------------------------------------------------------------------- keys: four threads a row
        const int tid = threadIdx.x - 128, key = tid >> 2, part = tid & 3;
        bool ok = true, more = walk.next(a, p);
        int t_in = 0, pos = 0, w = 0, off = 0, pid = -1, upto = 0;
        const int step_w = kKeys / a.page, step_off = kKeys - step_w * a.page;
        auto look_up = [&]() { pid = pos < upto ? a.table[p.b * a.table_stride + w] : -1; };
        auto begin_piece = [&]() {
            t_in = 0;
            upto = (int)min((int64_t)p.rg.total, (int64_t)p.rg.start + p.token + 1);
            pos = p.rg.first + p.r0 * kKeys + key;
            w = pos / a.page;
            off = pos - w * a.page;
            look_up();
        };
        if (more) begin_piece();
        // source of this thread's row of the next tile, which then moves on
        const uint8_t* src = nullptr;
        const float* scale_src = nullptr;
        bool full = false, dense = false;  // this thread's key exists; the tile is 32 rows of one page
        int row0 = 0;
        auto next_tile = [&]() {
            full = pid >= 0 && pid < a.P;
            dense = page_rows > 0 && full && pos - key + kKeys <= upto;
            row0 = pid * page_rows + off - key;
            const int64_t row = full ? pid * a.k_page + (int64_t)off * kJoint : 0;
            src = (const uint8_t*)a.k_pages + row * (E4M3 ? 1 : 2);
            if (E4M3) scale_src = a.k_scale + (full ? pid * a.ks_page + off : 0);
            pos += kKeys;
            w += step_w;
            off += step_off;
            if (off >= a.page) {
                off -= a.page;
                ++w;
            }
            if (++t_in < p.n) look_up();
            else if ((more = walk.next(a, p))) begin_piece();
        };
        // place in a stage of this row's 16-byte chunk 4 i + part: i even or odd, and (i / 2) kSub on
        const int row_at[2] = {key * 128 + ((part ^ (key & 7)) << 4), key * 128 + (((part + 4) ^ (key & 7)) << 4)};
        auto mark = [&](int st, bool here) {  // the tile's keys that exist
            const uint32_t bits = __ballot_sync(0xffffffffu, here);
            if (lane == 0) {
                uint32_t eight = 0;
#pragma unroll
                for (int k = 0; k < 8; ++k) eight |= ((bits >> (4 * k)) & 1u) << k;
                reinterpret_cast<uint8_t*>(s_valid + st)[warp - 4] = (uint8_t)eight;
            }
        };
        int T = 0;
        if constexpr (!E4M3) {
            // Two tiles' copies stay on their way while the next is fetched; where the ring is full they are handed over before
            // the wait for a stage.
            constexpr int kLag = 2;
            int sent = 0;
            auto hand_over = [&](int upto) {
                ptx::fence_proxy_async_smem();
                for (; sent < upto; ++sent) ptx::mbar_arrive(&k_full[sent % kRing]);
            };
            const uint32_t stages = ptx::smem_u32(smem + kK);
            for (; more && ok; ++T) {
                next_tile();
                const int st = T % kRing;
                if (!__all_sync(0xffffffffu, ptx::mbar_try_wait(&k_empty[st], ((T / kRing) & 1) ^ 1u))) {
                    copies_wait<0>();
                    hand_over(T);
                    ok = ptx::mbar_wait_bounded(&k_empty[st], ((T / kRing) & 1) ^ 1u, abort_flag, kWaitNs);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                if (dense) {  // the same for all threads: one fetches the tile, nine parts of 64 columns
                    copies_wait<0>();
                    hand_over(T);
                    if (tid == 0) {
                        s_valid[st] = 0xffffffffu;
                        ptx::mbar_expect_tx(&k_full[st], kStage);
#pragma unroll
                        for (int i = 0; i < kJoint / 64; ++i)
                            ptx::tma_load_2d(smem + kK + st * kStage + i * kSub, &tmap, i * 64, row0, &k_full[st]);
                    } else {
                        ptx::mbar_arrive(&k_full[st]);
                    }
                    ++sent;
                    continue;
                }
                mark(st, full);
                const uint32_t to[2] = {stages + st * kStage + row_at[0], stages + st * kStage + row_at[1]};
                const uint8_t* from = full ? src + part * 16 : (const uint8_t*)a.k_pages;
                if (full) {
#pragma unroll
                    for (int i = 0; i < kJoint / 32; ++i) copy16(to[i & 1] + (i >> 1) * kSub, from + i * 64, true);
                } else {
#pragma unroll
                    for (int i = 0; i < kJoint / 32; ++i) copy16(to[i & 1] + (i >> 1) * kSub, from, false);
                }
                copies_commit();
                if (T + 1 - sent > kLag) {
                    copies_wait<kLag>();
                    hand_over(T + 1 - kLag);
                }
            }
            copies_wait<0>();
            hand_over(T);
            if (tid == 0)
                for (int t = max(0, T - kRing); t < T; ++t) drain(&k_full[t % kRing], (t / kRing) & 1);
        } else {
            uint4 now[9], ahead[9];
            float scale_now = 0.f, scale_ahead = 0.f;
            bool full_ahead = false;
            auto fetch = [&]() {
                next_tile();
                full_ahead = full;
                scale_ahead = part == 0 && full ? *scale_src : 0.f;
#pragma unroll
                for (int i = 0; i < 9; ++i)
                    ahead[i] = full ? *reinterpret_cast<const uint4*>(src + (i * 4 + part) * 16) : make_uint4(0, 0, 0, 0);
            };
            bool loaded = more;
            if (more) fetch();
            for (; loaded && ok; ++T) {
                const bool here = full_ahead;
                scale_now = scale_ahead;
#pragma unroll
                for (int i = 0; i < 9; ++i) now[i] = ahead[i];
                loaded = more;
                if (more) fetch();
                const int st = T % kRing;
                ok = ptx::mbar_wait_bounded(&k_empty[st], ((T / kRing) & 1) ^ 1u, abort_flag, kWaitNs);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                mark(st, here);
                if (part == 0) {  // the scale, and its logarithm
                    s_scale[st * kKeys + key] = scale_now;
                    s_scale[(kRing + st) * kKeys + key] = __log2f(scale_now);
                }
#pragma unroll
                for (int i = 0; i < 9; ++i) {
                    uint8_t* sub = smem + kK + st * kStage + i * kSub + key * 128;  // 16 of the 64 columns of part i
                    const int ch0 = part * 2;
                    uint4 lo, hi;
                    e4m3x4_to_f16x4(now[i].x, lo.x, lo.y);
                    e4m3x4_to_f16x4(now[i].y, lo.z, lo.w);
                    e4m3x4_to_f16x4(now[i].z, hi.x, hi.y);
                    e4m3x4_to_f16x4(now[i].w, hi.z, hi.w);
                    *reinterpret_cast<uint4*>(sub + ((ch0 ^ (key & 7)) << 4)) = lo;
                    *reinterpret_cast<uint4*>(sub + (((ch0 + 1) ^ (key & 7)) << 4)) = hi;
                }
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(&k_full[st]);
            }
        }
        if (!ok && lane == 0) atomicCAS(error_flag, 0, (0x31 << 8) | 1);
    } else if (warp == 8) {
        // -------------------------------------------------------------------------------- products
        // The thread is chosen by elect.sync: a product of 32 columns was then measured at 16 cycles, and at 45 behind a test of
        // the lane.
        if (ptx::elect_one()) {
            constexpr uint32_t fmt = std::is_same<P, bf16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t kind = ~((1u << 7) | (1u << 10));
            constexpr uint32_t idesc_qk = (ptx::make_idesc_bf16(kRows, kKeys, false, false) & kind) | fmt;
            constexpr uint32_t idesc_pv = (ptx::make_idesc_bf16(kRows, kCols, false, true) & kind) | fmt;
            const uint64_t q_desc = ptx::make_smem_desc_sw128(ptx::smem_u32(smem + kQ), 16, 1024);
            const uint64_t k_desc = ptx::make_smem_desc_sw128(ptx::smem_u32(smem + kK), 16, 1024);
            const uint64_t v_desc = ptx::make_smem_desc_sw128(ptx::smem_u32(smem + kK), kSub, 1024);
            int T = 0, np = 0;
            bool ok = true;
            auto issue_values = [&](int t, bool add, int half) -> bool {
                if (!ptx::mbar_wait_bounded(&p_full[t & 1], (t >> 1) & 1, abort_flag, kWaitNs)) return false;
                ptx::tc_fence_after();
                const uint64_t vs = v_desc + (((t % kRing) * kStage + half * (kCols / 64) * kSub) >> 4);
#pragma unroll
                for (int k = 0; k < kKeys / 16; ++k)
                    ptx::mma_bf16_ts(tmem, tmem + kS + (t & 1) * kKeys + k * 8, vs + (k * 2048 >> 4), idesc_pv,
                                     add || k > 0);
                ptx::mma_commit(&k_empty[t % kRing]);
                ptx::mma_commit(&pv_done[t & 1]);
                return true;
            };
            while (ok && walk.next(a, p)) {
                ok = ptx::mbar_wait_bounded(q_full, np & 1, abort_flag, kWaitNs);
                ++np;
                for (int t = 0; t < p.n && ok; ++t, ++T) {
                    ok = ptx::mbar_wait_bounded(&k_full[T % kRing], (T / kRing) & 1, abort_flag, kWaitNs);
                    if (!ok) break;
                    ptx::tc_fence_after();
                    const uint64_t ks = k_desc + ((T % kRing) * kStage >> 4);
                    const uint32_t d = tmem + kS + (T & 1) * kKeys;
#pragma unroll
                    for (int k = 0; k < kJoint / 16; ++k) {
                        const uint64_t kd = ks + (((k >> 2) * kSub + (k & 3) * 32) >> 4);
                        if (k < kQTmem / 16) ptx::mma_bf16_ts(d, tmem + kQCol + k * 8, kd, idesc_qk, k > 0);
                        else ptx::mma_bf16_ss(d, q_desc + ((((k - kQTmem / 16) >> 2) * kQSub + (k & 3) * 32) >> 4), kd, idesc_qk, 1u);
                    }
                    ptx::mma_commit(&s_full[T & 1]);
                    if (t > 0) ok = issue_values(T - 1, t > 1, p.half);
                }
                if (ok) ok = issue_values(T - 1, p.n > 1, p.half);
            }
            if (!ok) atomicCAS(error_flag, 0, (0x32 << 8) | 1);
            ptx::mma_commit(drained);
            drain(drained, 0);
        }
    } else {
        // -------------------------------------------------------------------------------- softmax: a query row a thread
        const int r = threadIdx.x;
        const uint32_t my = tmem + ((uint32_t)(warp * 32) << 16);
        int T = 0, meetings = 0;
        bool ok = true;
        // values of tile t are added: a barrier for even and one for odd tiles, since a wait names a phase by its parity only
        // and the tile before may not be done either
        auto values_done = [&](int t) {
            return (bool)__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&pv_done[t & 1], (t >> 1) & 1, abort_flag, kWaitNs));
        };
        while (ok && walk.next(a, p)) {
            // The tile's queries [latent | rotary], zeros where it has no row: 64 columns at a time are copied to shared memory
            // by rows (eight threads a row); each thread takes its own row from there to tensor memory, the last three
            // parts stay.  Five parts first (two in spare buffers), then the other four.
            const bool real = r < p.rows;
            const int j = p.token, gr = p.row0 + r;
            const Q* q_base = (const Q*)a.q + p.b * a.q_b + j * a.q_s + (int64_t)(p.row0 - j * a.Hq) * a.q_h;
            const Q* q2_base = (const Q*)a.q2 + p.b * a.q2_b + j * a.q2_s + (int64_t)(p.row0 - j * a.Hq) * a.q2_h;
            auto buffer = [&](int i) { return i < 3 ? kQ + i * kQSub : kSpare + (i - 3) * kQSub; };
            auto fetch = [&](int part, int buf) {  // 64 columns
                const uint32_t to = ptx::smem_u32(smem + buffer(buf));
                const int ch = r & 7;
#pragma unroll
                for (int x = 0; x < kRows / 16; ++x) {
                    const int row = x * 16 + (r >> 3);
                    const Q* src = part < kLatent / 64 ? q_base + row * a.q_h + part * 64 : q2_base + row * a.q2_h;
                    const bool in = row < p.rows;
                    copy16(to + row * 128 + ((ch ^ (row & 7)) << 4), in ? (const void*)(src + ch * 8) : a.q, in);
                }
            };
            auto meet = [&]() -> bool {  // the four warps, bounded
                ptx::mbar_arrive(q_sync);
                const bool there = ptx::mbar_wait_bounded(q_sync, meetings++ & 1, abort_flag, kWaitNs);
                return (bool)__all_sync(0xffffffffu, there);
            };
            for (int part = 0; part < 5; ++part) fetch(part, part);
            copies_commit();
            float fac = fmaxf(fabsf(a.scale), 1e-30f) * kLog2e, up = 1.f;
            if (E4M3 && std::is_same<Q, bf16>::value) {  // the row's power of two (see the grouped form): a warp a row, 32 rows
                float mine = 0.f;
#pragma unroll 1
                for (int x0 = 0; x0 < 32; x0 += 8) {  // eight rows on their way at a time
                    uint4 u[8][3];
#pragma unroll
                    for (int x = 0; x < 8; ++x)
#pragma unroll
                        for (int c = 0; c < 3; ++c) {
                            const int row = warp * 32 + x0 + x, col = (c * 32 + lane) * 8;
                            u[x][c] = make_uint4(0, 0, 0, 0);
                            if (row < p.rows && col < kJoint)
                                u[x][c] = *reinterpret_cast<const uint4*>(col < kLatent ? q_base + row * a.q_h + col : q2_base + row * a.q2_h + col - kLatent);
                        }
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        float m = 0.f;
#pragma unroll
                        for (int c = 0; c < 3; ++c) {
                            const uint32_t w[4] = {u[x][c].x, u[x][c].y, u[x][c].z, u[x][c].w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float2 y = unpack2<Q>(w[i]);
                                m = fmaxf(m, fmaxf(fabsf(y.x), fabsf(y.y)));
                            }
                        }
                        m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m)));  // magnitudes order like their bits
                        if (lane == x0 + x) mine = m;
                    }
                }
                const int e = (__float_as_uint(mine) >> 23) & 255;
                const int field = e == 0 || e == 255 ? 127 : min(268 - e, 253);
                up = __uint_as_float((uint32_t)field << 23);
                fac *= __uint_as_float((uint32_t)(254 - field) << 23);
            }
            const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
            auto turn = [&](uint32_t u) -> uint32_t {
                u ^= sign;
                if (E4M3 && std::is_same<Q, bf16>::value) {
                    const float2 y = unpack2<Q>(u);
                    u = pack2<__half>(y.x * up, y.y * up);
                }
                return u;
            };
            auto chunk = [&](int buf, int i) { return reinterpret_cast<uint4*>(smem + buffer(buf) + r * 128 + ((i ^ (r & 7)) << 4)); };
            auto to_tmem = [&](int part, int buf) {
                uint32_t v[32];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 u = *chunk(buf, i);
                    v[4 * i] = turn(u.x);
                    v[4 * i + 1] = turn(u.y);
                    v[4 * i + 2] = turn(u.z);
                    v[4 * i + 3] = turn(u.w);
                }
                __syncwarp();
                ptx::tmem_st_32x32b_x32(my + kQCol + part * 32, v);
            };
            copies_wait<0>();
            if (!(ok = meet())) break;
#pragma unroll 1
            for (int part = 0; part < 5; ++part) to_tmem(part, part);
            if (!(ok = meet())) break;  // the buffers have been read
            fetch(5, 3);
            for (int part = 6; part < 9; ++part) fetch(part, part - 6);
            copies_commit();
            copies_wait<0>();
            if (!(ok = meet())) break;
            to_tmem(5, 3);
            if (sign || (E4M3 && std::is_same<Q, bf16>::value)) {
#pragma unroll 1
                for (int x = 0; x < 24; ++x) {
                    uint4* at = chunk(x >> 3, x & 7);
                    uint4 u = *at;
                    u.x = turn(u.x);
                    u.y = turn(u.y);
                    u.z = turn(u.z);
                    u.w = turn(u.w);
                    *at = u;
                }
            }
            __syncwarp();
            ptx::tmem_st_wait();
            ptx::tc_fence_before();
            ptx::fence_proxy_async_smem();
            ptx::mbar_arrive(q_full);

            float m = -INFINITY, mv = -INFINITY, l = 0.f;  // references of the sum and of the weighted values, in log2 units
            for (int t = 0; t < p.n; ++t, ++T) {
                const int st = T % kRing;
                ok = ptx::mbar_wait_bounded(&k_full[st], (T / kRing) & 1, abort_flag, kWaitNs) &&
                     ptx::mbar_wait_bounded(&s_full[T & 1], (T >> 1) & 1, abort_flag, kWaitNs);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ptx::tc_fence_after();
                uint32_t s[32];
                ptx::tmem_ld_32x32b_x32(my + kS + (T & 1) * kKeys, s);
                ptx::tmem_ld_wait();
                const uint32_t valid = s_valid[st];
                float x[32], lv[E4M3 ? 32 : 1];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(s[i]) * fac;
                if constexpr (E4M3) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 sc = *reinterpret_cast<const float4*>(s_scale + st * kKeys + i);
                        x[i] *= sc.x;
                        x[i + 1] *= sc.y;
                        x[i + 2] *= sc.z;
                        x[i + 3] *= sc.w;
                        const float4 lg = *reinterpret_cast<const float4*>(s_scale + (kRing + st) * kKeys + i);
                        lv[i] = lg.x;
                        lv[i + 1] = lg.y;
                        lv[i + 2] = lg.z;
                        lv[i + 3] = lg.w;
                    }
                }
                if (valid != 0xffffffffu) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (!((valid >> i) & 1)) x[i] = -INFINITY;
                }
                float t0 = -INFINITY, t1 = -INFINITY, v0 = -INFINITY, v1 = -INFINITY;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    t0 = fmaxf(t0, x[i]);
                    t1 = fmaxf(t1, x[i + 1]);
                    if constexpr (E4M3) {
                        v0 = fmaxf(v0, x[i] + lv[i]);
                        v1 = fmaxf(v1, x[i + 1] + lv[i + 1]);
                    }
                }
                // the values' reference stays within 2^118 of the sum's: keys of scale 0 may hold the largest scores alone, and 2^(m - mv)
                // below has to be finite (both references lag by up to 2^8)
                const float tm = fmaxf(t0, t1), tv = E4M3 ? fmaxf(fmaxf(v0, v1), tm - 118.f) : tm;
                if (tm > m + (m == -INFINITY ? 0.f : kGrow)) {
                    l *= m == -INFINITY ? 0.f : exp2f(m - tm);
                    m = tm;
                }
                const bool grow = tv > mv + (mv == -INFINITY ? 0.f : kGrow);
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = !grow ? 1.f : mv == -INFINITY ? 0.f : exp2f(mv - tv);
                    if (grow) mv = tv;
                    if (t > 0) {
                        ok = values_done(T - 1);
                        if (!ok) break;
                        ptx::tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < kCols; c += 32) {
                            uint32_t v[32];
                            ptx::tmem_ld_32x32b_x32(my + c, v);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                            ptx::tmem_st_32x32b_x32(my + c, v);
                        }
                    }
                }
                const float mz = m == -INFINITY ? 0.f : m, vz = mv == -INFINITY ? 0.f : mv;
                uint32_t pr[16];
                float l0 = 0.f, l1 = 0.f;
                // 8-bit: 2^(x + log2 scale - mv) = 2^(x - m) scale 2^(m - mv).  Every product is finite: mv is at least m - 126 and
                // x + log2 scale - 8.  What 2^(x - m) loses below 2^-126 would need values above 2^100 to be seen.
                const float g = E4M3 ? exp2f(mz - vz) : 1.f;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float e[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) e[k] = exp2f(x[i + k] - mz);
                    l0 += e[0] + e[2];
                    l1 += e[1] + e[3];
                    if constexpr (E4M3) {
                        const float4 sc = *reinterpret_cast<const float4*>(s_scale + st * kKeys + i);
                        e[0] = e[0] * sc.x * g;
                        e[1] = e[1] * sc.y * g;
                        e[2] = e[2] * sc.z * g;
                        e[3] = e[3] * sc.w * g;
                    }
                    pr[i / 2] = pack2<P>(e[0], e[1]);
                    pr[i / 2 + 1] = pack2<P>(e[2], e[3]);
                }
                l += l0 + l1;
                ptx::tmem_st_32x32b_x16(my + kS + (T & 1) * kKeys, pr);
                ptx::tmem_st_wait();
                ptx::tc_fence_before();
                ptx::mbar_arrive(&p_full[T & 1]);
            }
            if (ok) ok = values_done(T - 1);
            if (!ok) break;
            ptx::tc_fence_after();
            const int count = a.counts ? max(0, min(a.counts[p.b], a.S)) : a.S;
            const bool none = j >= count || l == 0.f;
            // a whole item is divided by its sum; a piece's values are brought to the units of its sum, 2^m
            float f = E4M3 ? (mv == -INFINITY ? 0.f : exp2f(mv - m)) : 1.f;
            if (p.whole) f = __fdividef(f, l);
            // pieces lie in groups of four columns, [column / 4][row][4]: a warp's 32 rows are one dense store
            const int64_t part0 = ((int64_t)blockIdx.x * 2 + (p.first ? 0 : 1)) * kRows;
            Q* out = (Q*)a.out + ((int64_t)p.b * a.S * a.Hq + gr) * kLatent + p.half * kCols;
#pragma unroll 1
            for (int c = 0; c < kCols; c += 32) {
                uint32_t v[32];
                __syncwarp();
                ptx::tmem_ld_32x32b_x32(my + c, v);
                ptx::tmem_ld_wait();
                if (!real) continue;
                if (p.whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float e[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) e[k] = none ? 0.f : __uint_as_float(v[i + k]) * f;
                        *reinterpret_cast<uint4*>(out + c + i) = Vec8<Q>::pack(e);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(part_o + part0 * kCols + ((c + i) / 4 * kRows + r) * 4) =
                            make_float4(__uint_as_float(v[i]) * f, __uint_as_float(v[i + 1]) * f, __uint_as_float(v[i + 2]) * f,
                                        __uint_as_float(v[i + 3]) * f);
                }
            }
            if (!p.whole && real) {
                part_ml[(part0 + r) * 2] = m;
                part_ml[(part0 + r) * 2 + 1] = l;
            }
            ptx::tc_fence_before();
        }
        if (!ok && lane == 0) atomicCAS(error_flag, 0, (0x33 << 8) | 1);
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    if (warp == 8) {
        __syncwarp();
        ptx::tmem_dealloc(tmem, 512);
    }
}
// Adds the pieces of an item, in their order along the keys: a lane a row.  One warp takes 32 rows and 32 columns or, where
// some item has many pieces, a block takes 32 rows and 8 columns and its warps every fourth piece.
template <typename T>
__global__ void __launch_bounds__(128) join_tiles_kernel(const AttnArgs a, int ctas, const int4* jobs, const float* part_ml,
                                                         const float* part_o) {
    __shared__ JobList list;
    __shared__ float4 s_o[4][2][32];
    __shared__ float2 s_ml[4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n_jobs = gather_jobs(list, ctas, jobs);
    const bool wide = list.most > 8;
    const int quads = wide ? 2 : 8, col_units = kCols / 4 / quads;
    constexpr int kRowUnits = kRows / 32;
    for (int u = wide ? blockIdx.x : blockIdx.x * 4 + warp; u < n_jobs * kRowUnits * col_units; u += wide ? gridDim.x : gridDim.x * 4) {
        const int jb = u / (kRowUnits * col_units), r = u / col_units % kRowUnits * 32 + lane, col = u % col_units * quads * 4;
        const int4 job = list.jobs[jb];
        int h, half, row0, rows;
        item_rows(a, job.y, kRows, h, half, row0, rows);
        float top = -INFINITY, sum = 0.f;
        float4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        // adds (m, l, values in units of 2^m); a piece without a finite score has seen nothing, or a NaN that its sum holds
        auto add = [&](float m, float l, const float4 (&o)[8]) {
            const float mn = fmaxf(top, m);
            const float f0 = top == -INFINITY ? 0.f : exp2f(top - mn), f1 = m == -INFINITY ? 0.f : exp2f(m - mn);
            sum = (top == -INFINITY ? sum : sum * f0) + (m == -INFINITY ? l : l * f1);
            top = mn;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                v[c].x = v[c].x * f0 + o[c].x * f1;
                v[c].y = v[c].y * f0 + o[c].y * f1;
                v[c].z = v[c].z * f0 + o[c].z * f1;
                v[c].w = v[c].w * f0 + o[c].w * f1;
            }
        };
        if (r < rows) {
#pragma unroll 2
            for (int i = wide ? warp : 0; i < job.z; i += wide ? 4 : 1) {
                const int64_t at = ((int64_t)(list.first[jb] + i) * 2 + (i == 0 ? job.w : 0)) * kRows;
                const float2 ml = *reinterpret_cast<const float2*>(part_ml + (at + r) * 2);
                const float4* src = reinterpret_cast<const float4*>(part_o + at * kCols) + col / 4 * kRows + r;
                float4 o[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) o[c] = c < quads ? src[c * kRows] : make_float4(0.f, 0.f, 0.f, 0.f);
                add(ml.x, ml.y, o);
            }
        }
        if (wide) {
            __syncthreads();  // the unit before has been read
            s_ml[warp][lane] = make_float2(top, sum);
            s_o[warp][0][lane] = v[0];
            s_o[warp][1][lane] = v[1];
            __syncthreads();
            if (warp > 0) continue;
#pragma unroll
            for (int x = 1; x < 4; ++x) {
                float4 o[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) o[c] = c < 2 ? s_o[x][c][lane] : make_float4(0.f, 0.f, 0.f, 0.f);
                add(s_ml[x][lane].x, s_ml[x][lane].y, o);
            }
        }
        if (r >= rows) continue;
        const int gr = row0 + r, count = a.counts ? max(0, min(a.counts[job.x], a.S)) : a.S;
        const bool none = gr / a.Hq >= count || sum == 0.f;
        const float inv = __fdividef(1.f, sum);
        T* out = (T*)a.out + ((int64_t)job.x * a.S * a.Hq + gr) * kLatent + half * kCols + col;
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
            if (c >= quads) break;
            float e[8] = {v[c].x, v[c].y, v[c].z, v[c].w, v[c + 1].x, v[c + 1].y, v[c + 1].z, v[c + 1].w};
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = none ? 0.f : e[k] * inv;
            *reinterpret_cast<uint4*>(out + c * 4) = Vec8<T>::pack(e);
        }
    }
}
}  // namespace tc

template <typename T, bool E4M3>
static void launch_latent_tc(AttnArgs a, int64_t B, const at::Tensor& q) {
    static std::atomic<uint64_t> done{0};
    allow_smem_once(tc::latent_tc_kernel<T, E4M3>, tc::kSmem, done);
    const int ctas = std::min(kMaxCtas, at::cuda::getCurrentDeviceProperties()->multiProcessorCount);
    a.halves = 2;
    a.cols = tc::kCols;
    a.token_tiles = (a.Hq + tc::kRows - 1) / tc::kRows;
    a.lead = 14;  // what an item costs besides its keys: queries 3 us, first keys 1.5 us, result 3 us; a round 0.6 us
    const int64_t items = (int64_t)a.S * a.token_tiles * a.halves;
    ATB_ARG(B * items * (ceil_div((int64_t)a.W * a.page, tc::kKeys) + 1 + a.lead) < (int64_t(1) << 31),
            "paged_latent_attention: too many sequences, query rows or positions for one call");
    const Workspace ws(q, ctas, tc::kRows, a.cols);
    cudaStream_t st = current_stream();
    int* error = gemm_error_flag(q.device()).data_ptr<int>();
    // whole tiles come by TMA where a tile cannot cross pages and pages lie a whole number of rows apart
    CUtensorMap tmap = {};
    int page_rows = 0;
    if (!E4M3 && a.page % tc::kKeys == 0 && a.k_page % kJoint == 0 && (int64_t)a.P * (a.k_page / kJoint) < (int64_t(1) << 31)) {
        page_rows = (int)(a.k_page / kJoint);
        tmap = make_tmap_bf16_public(a.k_pages, (int64_t)(a.P - 1) * page_rows + a.page, kJoint, kJoint, tc::kKeys);
    }
    tc::latent_tc_kernel<T, E4M3><<<ctas, tc::kThreads, tc::kSmem, st>>>(tmap, page_rows, a, (int)B, ws.jobs, ws.ml, ws.o, error);
    ATB_LAUNCH_CHECK();
    launch_behind(tc::join_tiles_kernel<T>, 4, st, a, ctas, (const int4*)ws.jobs, (const float*)ws.ml, (const float*)ws.o);
}

template <typename T, bool E4M3>
static void launch_latent(const AttnArgs& a, int64_t B, const at::Tensor& q) {
    // The tensor-core form from 33 heads on, where the other needs a second tile of 32 rows a token and with it the keys a
    // second time (89585 positions: 32 heads 47 us in one tile; 48 heads 78 us in two and 55 us here, 64 heads 80 and 56 us).
    // Several tokens of few heads stay with the other: here each token has tiles of its own.
    if (a.Hq > 32 && a.D1 == kLatent && a.D == kJoint) return launch_latent_tc<T, E4M3>(a, B, q);
    if (a.S * a.Hq <= 16) launch_latent_rows<T, E4M3, 1>(a, B, q);
    else launch_latent_rows<T, E4M3, 2>(a, B, q);
}

}  // namespace paged

using namespace paged;

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
    gemm_error_flag(q.device());  // made by the first call of either form, so that a later one can be captured
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
