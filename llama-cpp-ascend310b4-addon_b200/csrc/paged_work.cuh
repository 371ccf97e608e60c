// paged_work.cuh -- what the kernels that stream pages share: copies and
// tensor-core products of 16-bit pages with f32 operands.
#pragma once

#include <utility>

#include "common.cuh"
#include "paged_range.cuh"
#include "paged_store.cuh"

namespace b200 {

constexpr int kPaTok = 16;    // rows (positions, blocks) per unit
constexpr int kPaCtas = 148;  // CTAs of a full grid: one per SM

// Blocks of a sequence; a length outside the table is clamped.
__device__ __forceinline__ int paged_blocks(int len, int max_blocks, int page_size) {
    const unsigned b = len <= 0 ? 0u : ((unsigned)len + (unsigned)page_size - 1u) / (unsigned)page_size;
    return (int)min(b, (unsigned)max_blocks);
}

__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
// 16 bytes to dst + OFF.
template <int OFF>
__device__ __forceinline__ void pa_cp16_at(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
__device__ __forceinline__ void pa_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pa_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pa_ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The same at addr + OFF, and transposed.
template <int OFF>
__device__ __forceinline__ void pa_ldsm_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(OFF)
                 : "memory");
}
template <int OFF>
__device__ __forceinline__ void pa_ldsm_t_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(OFF)
                 : "memory");
}
template <bool BF16>
__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if (BF16)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from a zero accumulator.
template <bool BF16>
__device__ __forceinline__ void pa_mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if (BF16)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float pa_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// High 16-bit part of two values packed in a word; x, y become the remainders.
template <bool BF16>
__device__ __forceinline__ uint32_t pa_split(float& x, float& y) {
    const uint32_t w = pack16<BF16>(x, y);
    const float2 f = unpack16<BF16>(w);
    x -= f.x;
    y -= f.y;
    return w;
}

__device__ __forceinline__ float pa_warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// f(integral_constant<I>) for I of the sequence.
template <size_t... I, class F>
__device__ __forceinline__ void unrolled(std::index_sequence<I...>, F f) {
    (f(std::integral_constant<int, (int)I>{}), ...);
}

// p + I * step in one instruction.
template <int I>
__device__ __forceinline__ const uint8_t* pa_step(const uint8_t* p, uint32_t step) {
    if (I == 0) return p;
    uint64_t r;
    asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(step), "n"(I), "l"(p));
    return reinterpret_cast<const uint8_t*>(r);
}

}  // namespace b200
