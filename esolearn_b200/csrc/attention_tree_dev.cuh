// Device code shared by the tree attention kernels (attention_tree*.cu).
#pragma once

#include <cuda_fp16.h>

#include "attention_tree.cuh"
#include "mma_bf16.cuh"
#include "pipeline.cuh"

namespace sb {

constexpr float LOG2E = 1.4426950408889634f;

// mbar_wait (pipeline.cuh) with the clock looked at only after 256 failed polls:
// reading %globaltimer takes about 700 clocks, as long as the waits it bounds.
__device__ __forceinline__ bool mbar_wait_long(uint32_t bar, uint32_t parity) {
    uint64_t t0 = 0;
    for (uint32_t it = 1;; it++) {
        uint32_t done;
        asm volatile(
            "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if ((it & 255) == 0) {
            const uint64_t t = global_ns();
            if (t0 == 0) t0 = t;
            else if (t - t0 > SB_WAIT_NS) return false;
        }
    }
}

// Asynchronous copies of which the first n bytes are read and the rest is zero.
__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async4_fill(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_rna(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// x, y as TERMS pairs of 16-bit terms: x = sum of the low halves.
template <int TERMS>
__device__ __forceinline__ void split_bf16x2(float x, float y, uint32_t (&o)[TERMS]) {
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        o[t] = *reinterpret_cast<const uint32_t *>(&h);
        if (t + 1 < TERMS) x = __fsub_rn(x, __uint_as_float(o[t] << 16)), y = __fsub_rn(y, __uint_as_float(o[t] & 0xffff0000u));
    }
}
template <int TERMS>
__device__ __forceinline__ void split_f16x2(float x, float y, uint32_t (&o)[TERMS]) {
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
        const __half2 h = __floats2half2_rn(x, y);
        o[t] = *reinterpret_cast<const uint32_t *>(&h);
        if (t + 1 < TERMS) {
            const float2 f = __half22float2(h);
            x = __fsub_rn(x, f.x), y = __fsub_rn(y, f.y);
        }
    }
}

// Two int8 codes (bytes sel of w, offset by 128) as exact f16: 0x6400 | byte is
// 1024 + byte, and 1024 + code + 128 - 1152 = code.
__device__ __forceinline__ uint32_t code2_f16(uint32_t w, uint32_t sel) {
    uint32_t r = __byte_perm(w, 0x64646464u, sel);
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&r), off);
    return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ unsigned long long low_bits(long long n) {
    return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}
// Bits of positions base .. base+63 that token i sees (bit n: position base + n); of the tokens only the first n_vis are
// there to be seen (the others do not exist, have no place in the table, or lie behind all rows of the CTA).
__device__ __forceinline__ unsigned long long visible_bits(const TreeAttnArgs &a, int b, int i, long long ctx, int n_vis,
                                                           long long base) {
    const long long j0 = base - ctx;  // token index of bit 0 (negative: context)
    unsigned long long w = low_bits(-j0);
    if (i < 0) return w;
    if (!a.mask) {
        w |= low_bits((long long)min(i + 1, n_vis) - j0);
    } else {
        const unsigned long long *row = a.mask + (size_t)b * a.mask_ld + (size_t)i * a.mask_words;
        unsigned long long m = 0;
        if (j0 < 0) {
            if (j0 > -64) m = __ldg(row) << (int)(-j0);
        } else {
            const int k = (int)(j0 >> 6), s = (int)(j0 & 63);
            if (k < a.mask_words) m = __ldg(row + k) >> s;
            if (s && k + 1 < a.mask_words) m |= __ldg(row + k + 1) << (64 - s);
        }
        w |= m & low_bits((long long)n_vis - j0);
    }
    return w;
}

// A box of a [rows][hd] tensor map from element x of row y on (no multicast);
// rows behind the tensor's end are zeros.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// A query row's elements x, of which the four lanes of a group hold a quarter
// each, as f16 terms: scale is 2^-e with e the exponent of the row's largest
// finite element (held to where 2^e and 2^-e are normal), f = 2^e * log2(e).
template <int N>
__device__ __forceinline__ void row_exponent(const float (&x)[N], float &scale, float &f) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float y = fabsf(x[i]);
        if (y < INFINITY) m = fmaxf(m, y);
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const int e = min(max((int)(__float_as_uint(m) >> 23), 2), 252);
    scale = __uint_as_float((uint32_t)(254 - e) << 23);
    f = LOG2E * __uint_as_float((uint32_t)e << 23);
}

// Four elements of an output row: x / l (0 where nothing was seen, or the token does not exist).
template <int HD, bool BF16>
__device__ __forceinline__ void tree_store4(const TreeAttnArgs &a, int b, int g, int row, int d, float4 x, float l, int n_new) {
    const int t = row / a.rep, h = row - t * a.rep;
    const size_t at = ((size_t)((size_t)b * a.T + t) * a.n_heads + (size_t)(g * a.rep + h)) * HD + d;
    const float k = l == 0.0f ? 0.0f : 1.0f / l;
    x.x *= k, x.y *= k, x.z *= k, x.w *= k;
    if (l == 0.0f || t >= n_new) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (BF16) {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y), z = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(a.out) + at) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&y), *reinterpret_cast<const uint32_t *>(&z));
    } else {
        *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = x;
    }
}

// The end of a CTA that holds `rows` (of ROWS) query rows from row0 on: its PARTS
// position groups' unnormalised outputs red [PARTS][ROWS][HD] with maxima rm and
// sums rl [PARTS][ROWS] are joined in order, to the output or, with several
// splits, to the workspace, from where tree_join_kernel takes them.
template <int HD, bool BF16, int PARTS, int ROWS, int THREADS>
__device__ __forceinline__ void tree_finish(const TreeAttnArgs &a, const float *red, const float *rm, const float *rl, int rows,
                                            int row0, int b, int g, int n_new, int split, size_t tile) {
    const size_t first = (tile * a.n_splits + split) * ROWS;
    for (int i = threadIdx.x; i < rows * (HD / 4); i += THREADS) {
        const int r = i / (HD / 4), d = (i - r * (HD / 4)) * 4;
        float M = -INFINITY, L = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < PARTS; w++) M = fmaxf(M, rm[w * ROWS + r]);
#pragma unroll
        for (int w = 0; w < PARTS; w++) {
            const float mw = rm[w * ROWS + r];
            if (mw == -INFINITY && rl[w * ROWS + r] == 0.0f) continue;
            const float f = ex2(mw - M);
            const float4 y = *reinterpret_cast<const float4 *>(red + (size_t)(w * ROWS + r) * HD + d);
            L = fmaf(rl[w * ROWS + r], f, L);
            x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
        }
        if (a.n_splits == 1) {
            tree_store4<HD, BF16>(a, b, g, row0 + r, d, x, L, n_new);
        } else {
            *reinterpret_cast<float4 *>(a.part + (first + r) * HD + d) = x;
            if (d == 0) a.ml[first + r] = make_float2(M, L);
        }
    }
}

}  // namespace sb
