// SPDX-License-Identifier: Apache-2.0
// What the kernels of the paged generation cache share: the layout of a cache, 16-byte vectors of its element types and
// the argument checks of their entry points.
//
// A cache is `pages [P, H, page, D]` (inner three dimensions dense): page p holds `page` consecutive positions of one
// sequence for every head.  Its elements are those of the model (bf16 / fp16), or e4m3 with one fp32 scale per (position,
// head) in `scale [P, H, page]`.  `table [B, W]` names the pages of each sequence in order; a page id outside [0, P) holds
// nothing: writes to it are dropped, reads skip it.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace atb {
namespace paged {

constexpr float kE4M3Max = 448.f;
constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100: rows below this are quantised as if this were their largest value

template <typename T>
struct Vec8;  // eight 16-bit elements of one 16-byte access
template <>
struct Vec8<bf16> {
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        unpack8(*reinterpret_cast<const bf16x8*>(&u), f);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        const bf16x8 p = pack8(f);
        return *reinterpret_cast<const uint4*>(&p);
    }
};
template <>
struct Vec8<__half> {
    static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
        const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(h[i]);
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
        uint4 u;
        __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        return u;
    }
};

// two e4m3 values (low byte first) as fp16, exactly
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n" : "=r"(r) : "r"(two));
    return r;
}
// four e4m3 values: the low two and the high two
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}\n"
        : "=r"(lo), "=r"(hi) : "r"(four));
}
__device__ __forceinline__ void unpack_e4m3x8(const uint2& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t h = e4m3x2_to_f16x2(w[i]);
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
// eight fp32 values as e4m3, to nearest, saturating at 448 (NaN stays NaN)
__device__ __forceinline__ uint2 pack_e4m3x8(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(f[2 * i + 1]), "f"(f[2 * i]));
        w[i] = r;
    }
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}
// maximum that keeps a NaN, so that a row with one gets a NaN scale
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float e4m3_scale(float amax) { return __fdiv_rn(max_nan(amax, kTiny), kE4M3Max); }

// ---- host side ------------------------------------------------------------------------------------------------------
#define ATB_ARG(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

inline bool is_e4m3(const at::Tensor& t) { return t.scalar_type() == at::kFloat8_e4m3fn; }

// whether every slice along the first dimension is dense (a dimension of one element may have any stride)
inline bool dense_inside(const at::Tensor& t) {
    int64_t step = 1;
    for (int64_t i = t.dim() - 1; i > 0; --i) {
        if (t.size(i) != 1 && t.stride(i) != step) return false;
        step *= t.size(i);
    }
    return true;
}

// a cache tensor: device, layout, type against the inputs' type, scales when its elements are e4m3
inline void check_pages(const char* op, const at::Tensor& pages, const c10::optional<at::Tensor>& scale, const at::Tensor& x) {
    ATB_ARG(pages.dim() == 4, op, ": pages must be [pages, heads, page, dim]");
    ATB_ARG(pages.size(2) > 0, op, ": a page holds at least one position");
    ATB_ARG(pages.device() == x.device(), op, ": all tensors must be on one device");
    ATB_ARG(dense_inside(pages), op, ": the heads, positions and elements of a page must be dense");
    ATB_ARG((reinterpret_cast<uintptr_t>(pages.data_ptr()) & 15) == 0 && (pages.stride(0) * pages.element_size()) % 16 == 0,
            op, ": pages must be 16-byte aligned");
    if (is_e4m3(pages)) {
        ATB_ARG(scale.has_value(), op, ": an e4m3 cache needs its scales");
        ATB_ARG(scale->scalar_type() == at::kFloat && scale->dim() == 3 && scale->size(0) == pages.size(0) &&
                    scale->size(1) == pages.size(1) && scale->size(2) == pages.size(2),
                op, ": scales must be fp32 [pages, heads, page]");
        ATB_ARG(dense_inside(*scale), op, ": the scales of a page must be dense");
        ATB_ARG(scale->device() == x.device(), op, ": all tensors must be on one device");
    } else {
        ATB_ARG(!scale.has_value(), op, ": scales belong to an e4m3 cache");
    }
}

inline void check_table(const char* op, const at::Tensor& table, const at::Tensor& lens, const c10::optional<at::Tensor>& counts,
                        const at::Tensor& pages, int64_t B) {
    ATB_ARG(table.dim() == 2 && table.size(0) == B && table.scalar_type() == at::kInt, op, ": page_table must be int32 [batch, pages]");
    ATB_ARG(table.size(1) <= 1 || table.stride(1) == 1, op, ": the rows of page_table must be dense");
    ATB_ARG(lens.dim() == 1 && lens.size(0) == B && lens.scalar_type() == at::kInt && lens.is_contiguous(), op,
            ": starts / lengths must be dense int32 [batch]");
    ATB_ARG(table.device() == pages.device() && lens.device() == pages.device(), op, ": all tensors must be on one device");
    if (counts.has_value())
        ATB_ARG(counts->dim() == 1 && counts->size(0) == B && counts->scalar_type() == at::kInt && counts->is_contiguous() &&
                    counts->device() == pages.device(),
                op, ": counts must be dense int32 [batch]");
    ATB_ARG(table.size(1) * pages.size(2) < (int64_t(1) << 31) - (1 << 20), op, ": a sequence holds fewer than 2^31 positions");
}

// [..., D] rows as the kernels read them: dense, 16-byte aligned elements; other layouts are copied
inline at::Tensor rows16(const at::Tensor& t) {
    bool ok = t.stride(-1) == 1 && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
    for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) * t.element_size()) % 16 == 0);
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

template <typename P>
inline P* ptr(const c10::optional<at::Tensor>& t) {
    return t.has_value() ? reinterpret_cast<P*>(t->data_ptr()) : nullptr;
}

}  // namespace paged
}  // namespace atb
