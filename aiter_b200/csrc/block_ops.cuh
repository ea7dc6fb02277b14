// What stands between two GEMMs of a transformer block, one kernel launch each, forward only:
//
//   gated_residual_norm   u = x | norm(x) * post_weight + post_bias
//                         h = residual_scale * residual + gate * u
//                         y = norm(h) * (weight_offset + weight) + bias
//                         norm(v) = v * rsqrt(mean v^2 + eps)  or  (v - mean v) * rsqrt(mean (v - mean v)^2 + eps)
//   act_and_mul           y[:, j] = act(in[:, j]) * in[:, n + j]
//
// y leaves as bf16 / fp16 / fp32, or as the operand of an MX GEMM: e4m3 or packed e2m1 with one UE8M0 scale per 32
// elements in the layout the GEMM reads (the arithmetic and layouts of quant_mx.cuh, applied to the fp32 values: the
// 16-bit rounding between a norm and a separate quantiser is left out).  All sums and the residual sum h are held in
// fp32; y is computed from h before h is rounded to its stored type.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cstdint>
#include "activation.cuh"
#include "gemm_common.cuh"
#include "quant_mx.cuh"

namespace b200 {

// element types of row tensors and parameters: OUT_BF16 / OUT_F16 / OUT_F32, y also OUT_E2M1 / OUT_MXFP8 (here: one scale
// per 32 elements)
struct RowTensor
{
    void* ptr;
    long long ld; // elements between rows
    int dt;
};
// A parameter of a row: [n] (ld 0), or [groups, n] where row r reads entry r / rows_per
struct RowParam
{
    const void* ptr;
    long long ld;
    int dt;
    unsigned rows_per;
};

struct BlockScales
{
    uint8_t* ptr;
    int cols;   // columns of the scale array
    int layout; // QuantScaleLayout
};

struct NormParams
{
    RowTensor x, res, h, y; // res.ptr null: no residual; h.ptr null: h is not stored
    RowParam weight, bias, gate, post_weight, post_bias;
    int gate_scalar;        // the gate is one value per entry
    int post;               // 1: the first norm is applied
    int layer;              // 0 rms, 1 layer norm
    float res_scale, weight_offset, eps, inv_n;
    unsigned M, n;
    BlockScales sf;
};

__device__ __forceinline__ float dec16(uint32_t bits, int dt)
{
    return dt == OUT_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

__device__ __forceinline__ float load_elem_any(const void* base, int dt, size_t at)
{
    return dt == OUT_F32 ? static_cast<const float*>(base)[at] : dec16(static_cast<const uint16_t*>(base)[at], dt);
}
__host__ __device__ constexpr int bytes_of_mode(int dt) { return dt == OUT_F32 ? 4 : dt == OUT_E2M1 || dt == OUT_MXFP8 ? 1 : 2; }

// ---- raw vectors: VEC = 8 elements as one or two 16-byte loads, VEC = 1 one element
template <int VEC, bool B32>
struct Raw
{
    uint32_t w[VEC == 1 ? 1 : (B32 ? 8 : 4)];
};
// rows are read once: keep them out of the way of the parameters, which every row of an SM reads again, in L1
__device__ __forceinline__ uint4 ld_stream16(const void* p)
{
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
template <int VEC, bool B32>
__device__ __forceinline__ void ld_raw(Raw<VEC, B32>& r, const void* base, size_t at)
{
    if(VEC == 1)
        r.w[0] = B32 ? static_cast<const uint32_t*>(base)[at] : static_cast<const uint16_t*>(base)[at];
    else
    {
        const uint8_t* p = static_cast<const uint8_t*>(base) + at * (B32 ? 4 : 2);
#pragma unroll
        for(int i = 0; i < (B32 ? 2 : 1); ++i)
        {
            const uint4 v    = ld_stream16(p + 16 * i);
            r.w[VEC == 1 ? 0 : 4 * i]     = v.x;
            r.w[VEC == 1 ? 0 : 4 * i + 1] = v.y;
            r.w[VEC == 1 ? 0 : 4 * i + 2] = v.z;
            r.w[VEC == 1 ? 0 : 4 * i + 3] = v.w;
        }
    }
}
template <int VEC, bool B32>
__device__ __forceinline__ void unpack(const Raw<VEC, B32>& r, int dt, float (&v)[VEC])
{
    if(B32)
    {
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            v[i] = __uint_as_float(r.w[VEC == 1 ? 0 : i]);
    }
    else if(VEC == 1)
        v[0] = dec16(r.w[0], dt);
    else if(dt == OUT_BF16)
    {
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            v[i] = __uint_as_float((i & 1) ? (r.w[VEC == 1 ? 0 : i >> 1] & 0xFFFF0000u) : (r.w[VEC == 1 ? 0 : i >> 1] << 16));
    }
    else
    {
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            v[i] = dec16((r.w[VEC == 1 ? 0 : i >> 1] >> (16 * (i & 1))) & 0xFFFFu, OUT_F16);
    }
}
// parameters: the type is looked at here (they are few, and in L1 after the first rows).  Plain loads: a gate or a modulation may
// come from the kernel just before, which this one overlaps up to its dependency wait.
template <int VEC>
__device__ __forceinline__ void ld_param(const void* base, int dt, size_t at, float (&v)[VEC])
{
    if(VEC == 1)
        v[0] = dt == OUT_F32 ? static_cast<const float*>(base)[at] : dec16(static_cast<const uint16_t*>(base)[at], dt);
    else if(dt == OUT_F32)
    {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
#pragma unroll
        for(int i = 0; i < VEC / 4; ++i)
        {
            const float4 t = p[i];
            v[VEC == 1 ? 0 : 4 * i]     = t.x;
            v[VEC == 1 ? 0 : 4 * i + 1] = t.y;
            v[VEC == 1 ? 0 : 4 * i + 2] = t.z;
            v[VEC == 1 ? 0 : 4 * i + 3] = t.w;
        }
    }
    else
    {
        const uint4 t = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at);
        Raw<8, false> r;
        r.w[0] = t.x, r.w[1] = t.y, r.w[2] = t.z, r.w[3] = t.w;
        float f[8];
        unpack<8, false>(r, dt, f);
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            v[i] = f[i];
    }
}
template <int VEC>
__device__ __forceinline__ void st_vec(void* base, int dt, size_t at, const float (&v)[VEC])
{
    if(VEC == 1)
        store_out(base, at, v[0], dt);
    else if(dt == OUT_F32)
    {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
#pragma unroll
        for(int i = 0; i < VEC / 4; ++i)
            p[i] = make_float4(v[VEC == 1 ? 0 : 4 * i], v[VEC == 1 ? 0 : 4 * i + 1], v[VEC == 1 ? 0 : 4 * i + 2], v[VEC == 1 ? 0 : 4 * i + 3]);
    }
    else
    {
        const bool f16 = (dt == OUT_F16);
        uint32_t w[4];
#pragma unroll
        for(int i = 0; i < 4; ++i)
            w[i] = pack_out16x2(v[VEC == 1 ? 0 : 2 * i], v[VEC == 1 ? 0 : 2 * i + 1], f16);
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Eight elements on any element's address: the 16-byte pieces that hold those of them that are wanted, lo .. hi - 1 (no other piece is
// read: a piece with one byte of a tensor lies in its memory), and how far the first one stands from its piece's beginning.
template <bool B32>
struct Pieces
{
    uint32_t w[B32 ? 12 : 8];
};
template <bool B32>
__device__ __forceinline__ int shift_of(const void* p) // of every group of eight of a row
{
    return static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / (B32 ? 4 : 2);
}
template <bool B32>
__device__ __forceinline__ void ld_pieces(Pieces<B32>& r, const uint8_t* p, int s, int lo, int hi)
{
    const uint4* piece = reinterpret_cast<const uint4*>(p - s * (B32 ? 4 : 2));
    auto take          = [&](int i, bool wanted) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if(wanted)
            v = piece[i]; // (through L1: the next thread reads one of the pieces too)
        r.w[4 * i] = v.x, r.w[4 * i + 1] = v.y, r.w[4 * i + 2] = v.z, r.w[4 * i + 3] = v.w;
    };
    if(B32)
    {
        take(0, lo < 4 - s);
        take(1, hi > 4 - s && lo < 8 - s);
        take(B32 ? 2 : 0, hi > 8 - s);
    }
    else
    {
        take(0, lo < 8 - s);
        take(1, hi > 8 - s);
    }
}
// moved into place
template <bool B32>
__device__ __forceinline__ void align_pieces(Raw<8, B32>& r, Pieces<B32> q, int s)
{
    if(s != 0) // (the same for a whole row)
    {
        if(B32)
        {
            // by two words, by one
#pragma unroll
            for(int i = 0; i < 9; ++i)
                q.w[B32 ? i : 0] = (s & 2) ? q.w[B32 ? i + 2 : 0] : q.w[B32 ? i : 0];
#pragma unroll
            for(int i = 0; i < 8; ++i)
                q.w[i] = (s & 1) ? q.w[B32 ? i + 1 : 0] : q.w[i];
        }
        else
        {
            // by two words, by one, by half a word
#pragma unroll
            for(int i = 0; i < 6; ++i)
                q.w[i] = (s & 4) ? q.w[i + 2] : q.w[i];
#pragma unroll
            for(int i = 0; i < 5; ++i)
                q.w[i] = (s & 2) ? q.w[i + 1] : q.w[i];
#pragma unroll
            for(int i = 0; i < 4; ++i)
                q.w[i] = __funnelshift_r(q.w[i], q.w[i + 1], (s & 1) * 16);
        }
    }
#pragma unroll
    for(int i = 0; i < (B32 ? 8 : 4); ++i)
        r.w[i] = q.w[i];
}
// a parameter's values, whose type is looked at here
__device__ __forceinline__ void ld_param_shifted(const void* base, int dt, long long at, int lo, int hi, float (&v)[8])
{
    auto go = [&](auto b32) {
        constexpr bool B32 = decltype(b32)::value;
        const uint8_t* p   = static_cast<const uint8_t*>(base) + at * (B32 ? 4 : 2);
        const int s        = shift_of<B32>(p);
        Pieces<B32> q;
        ld_pieces<B32>(q, p, s, lo, hi);
        Raw<8, B32> r;
        align_pieces<B32>(r, q, s);
        unpack<8, B32>(r, dt, v);
    };
    if(dt == OUT_F32)
        go(std::true_type{});
    else
        go(std::false_type{});
}
// elements `lo` .. `hi` - 1 of the eight that begin at element `at`
__device__ __forceinline__ void st_shifted(void* base, int dt, long long at, int lo, int hi, const float (&v)[8])
{
    uint8_t* p = static_cast<uint8_t*>(base) + at * (dt == OUT_F32 ? 4 : 2);
    if(hi - lo == 8 && (reinterpret_cast<uintptr_t>(p) & 15) == 0)
        st_vec<8>(p, dt, 0, v);
    else
#pragma unroll
        for(int i = 0; i < 8; ++i)
            if(i >= lo && i < hi)
                store_out(p, i, v[i], dt);
}

// largest magnitude of three values; a NaN among them survives
__device__ __forceinline__ float amax3(float a, float b, float c)
{
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// UE8M0 byte of a block with largest magnitude `ab` (bits, sign-less): the exponent of ab / max_pos rounded up.  With
// max_pos = 1.75 * 2^8 (e4m3) or 1.5 * 2^2 (e2m1) the division only decides whether the significand of ab is above that of
// max_pos - the two floats around a significand of 1.75 or 1.5 divide to values on their own side of 1 -, so for normal quotients
// one addition carries into the exponent.  Zero, quotients below the normal range, infinity and NaN take the division itself.
template <bool FP4>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t ab)
{
    if(ab - (16u << 23) < (0x7F800000u - (16u << 23)))
        return ((ab + (FP4 ? 0x3FFFFFu : 0x1FFFFFu)) >> 23) - (FP4 ? 2u : 8u);
    const uint32_t qb = __float_as_uint(__fdiv_rn(__uint_as_float(ab), FP4 ? 6.0f : 448.0f));
    const uint32_t ex = (qb >> 23) & 0xFFu;
    return ex + (((qb & 0x7FFFFFu) != 0u && ex < 0xFFu) ? 1u : 0u);
}

// ---- one 32-element block held by four neighbouring lanes, eight values each
// Returns the UE8M0 byte (the same in the four lanes); q: 8 e4m3 bytes in q[0..1], or 8 e2m1 codes in q[0].
template <bool FP4>
__device__ __forceinline__ uint32_t mx_block(const float (&v)[8], uint32_t (&q)[2])
{
    const float m = amax3(amax3(v[0], v[1], v[2]), amax3(v[3], v[4], v[5]), amax3(v[6], v[7], v[7]));
    // (the integer order of sign-less bit patterns is the order of the values with NaN on top)
    uint32_t ab = __float_as_uint(m);
    ab          = max(ab, __shfl_xor_sync(0xffffffffu, ab, 1));
    ab          = max(ab, __shfl_xor_sync(0xffffffffu, ab, 2));
    const uint32_t byte = mx_scale_byte<FP4>(ab);
    const float rscale  = __uint_as_float(byte == 0xFFu ? 0x7F800001u : (byte == 254u ? 0x00400000u : ((254u - byte) << 23)));
    const float2 r2     = make_float2(rscale, rscale);
    float2 z[4];
#pragma unroll
    for(int i = 0; i < 4; ++i)
        z[i] = __fmul2_rn(make_float2(v[2 * i], v[2 * i + 1]), r2);
    if(FP4)
    {
        uint32_t packed = 0;
#pragma unroll
        for(int i = 0; i < 4; ++i)
            packed |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(z[i], __NV_E2M1, cudaRoundNearest)) << (8 * i);
        q[0] = packed;
        q[1] = 0;
    }
    else
    {
#pragma unroll
        for(int h = 0; h < 2; ++h)
        {
            const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(z[2 * h], __NV_SATFINITE, __NV_E4M3);
            const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(z[2 * h + 1], __NV_SATFINITE, __NV_E4M3);
            q[h] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
        }
    }
    return byte;
}

// byte position of (row, block) in a scale array
__device__ __forceinline__ size_t sf_offset(const BlockScales& sf, unsigned row, unsigned kb)
{
    if(sf.layout == QSL_E8M0_SHUFFLE)
        return static_cast<size_t>(row >> 5) * (static_cast<size_t>(sf.cols) * 32) + (kb >> 3) * 256u + (kb & 3) * 64u + (row & 15) * 4u + ((kb >> 2) & 1) * 2u + ((row >> 4) & 1);
    if(sf.layout == QSL_M32K4)
        return static_cast<size_t>(row >> 5) * (static_cast<size_t>(sf.cols) * 32) + (kb >> 2) * 128u + (row & 31) * 4u + (kb & 3);
    return static_cast<size_t>(row) * sf.cols + kb;
}
// What the quantiser leaves around the blocks: the scale columns behind K (e8m0_shuffle rounds them up to 8) and the rows
// behind M of the last group of 32.  Called by the `threads` threads that own row `row`.
__device__ __forceinline__ void fill_scale_padding(const BlockScales& sf, unsigned row, unsigned M, unsigned kblocks, unsigned t, unsigned threads)
{
    if(sf.layout == QSL_PLAIN)
        return;
    const uint8_t fill  = sf.layout == QSL_M32K4 ? 0x7F : 0;
    const unsigned cols = sf.layout == QSL_E8M0_SHUFFLE ? (kblocks + 7) / 8 * 8 : kblocks;
    for(unsigned kb = kblocks + t; kb < cols; kb += threads)
        sf.ptr[sf_offset(sf, row, kb)] = fill;
    if(row == M - 1)
        for(unsigned r = M; r < (M + 31) / 32 * 32; ++r)
            for(unsigned kb = t; kb < cols; kb += threads)
                sf.ptr[sf_offset(sf, r, kb)] = fill;
}

__device__ __forceinline__ float warp_sum(float v, unsigned lanes = 32)
{
#pragma unroll
    for(unsigned d = 16; d > 0; d >>= 1)
        if(d < lanes)
            v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Sum over the threads of a row: 8, 16 or 32 lanes, or the whole CTA (`slot`: consecutive sums use different slots, so that one
// barrier a sum is enough).  The order of the additions is fixed.
__device__ __forceinline__ float row_sum(float v, float (*red)[32], int slot)
{
    v = warp_sum(v, blockDim.x);
    if(blockDim.x <= 32)
        return v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if(lane == 0)
        red[slot][warp] = v;
    __syncthreads();
    return warp_sum(lane < static_cast<int>(blockDim.x >> 5) ? red[slot][lane] : 0.f);
}

// One row of y: eight values (VEC = 8) or one at column `col`
template <int VEC>
__device__ __forceinline__ void emit(const NormParams& prm, unsigned row, unsigned col, bool in, const float (&y)[VEC])
{
    if(VEC == 8 && prm.y.dt >= OUT_E2M1)
    {
        float f[8];
#pragma unroll
        for(int i = 0; i < 8; ++i)
            f[i] = y[VEC == 1 ? 0 : i];
        uint32_t q[2], byte;
        uint8_t* dst = static_cast<uint8_t*>(prm.y.ptr) + static_cast<size_t>(row) * prm.y.ld;
        if(prm.y.dt == OUT_E2M1)
        {
            byte = mx_block<true>(f, q);
            if(in)
                *reinterpret_cast<uint32_t*>(dst + (col >> 1)) = q[0];
        }
        else
        {
            byte = mx_block<false>(f, q);
            if(in)
                *reinterpret_cast<uint2*>(dst + col) = make_uint2(q[0], q[1]);
        }
        if(prm.sf.layout == QSL_M32K4)
        {
            // four neighbouring blocks of a row are four neighbouring bytes: one word per 16 lanes
            byte |= __shfl_down_sync(0xffffffffu, byte, 4) << 8;
            byte |= __shfl_down_sync(0xffffffffu, byte, 8) << 16;
            if(in && (threadIdx.x & 15) == 0)
                *reinterpret_cast<uint32_t*>(prm.sf.ptr + sf_offset(prm.sf, row, col >> 5)) = byte;
        }
        else if(in && (threadIdx.x & 3) == 0)
            prm.sf.ptr[sf_offset(prm.sf, row, col >> 5)] = static_cast<uint8_t>(byte);
    }
    else if(in)
        st_vec<VEC>(prm.y.ptr, prm.y.dt, static_cast<size_t>(row) * prm.y.ld + col, y);
}

__device__ __forceinline__ size_t param_at(const RowParam& p, unsigned row) { return p.ld == 0 ? 0 : static_cast<size_t>(row / p.rows_per) * p.ld; }

// h of VEC columns from x's (already normed if there is a first norm) and the residual's values.  get(parameter, at, v): the
// parameter's values of these columns, its entry beginning at element `at`.
template <int VEC, typename Get>
__device__ __forceinline__ void residual_sum(const NormParams& prm, Get&& get, size_t at_pw, size_t at_pb, size_t at_g, float gate1, float mean, float rstd,
                                             bool has_res, const float (&res)[VEC], float (&h)[VEC])
{
    if(prm.post)
    {
        float w[VEC];
        if(prm.post_weight.ptr != nullptr)
            get(prm.post_weight, at_pw, w);
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            h[i] = (h[i] - mean) * rstd * (prm.post_weight.ptr != nullptr ? w[i] : 1.f);
        if(prm.post_bias.ptr != nullptr)
        {
            get(prm.post_bias, at_pb, w);
#pragma unroll
            for(int i = 0; i < VEC; ++i)
                h[i] += w[i];
        }
    }
    if(prm.gate.ptr != nullptr)
    {
        if(prm.gate_scalar)
        {
#pragma unroll
            for(int i = 0; i < VEC; ++i)
                h[i] *= gate1;
        }
        else
        {
            float g[VEC];
            get(prm.gate, at_g, g);
#pragma unroll
            for(int i = 0; i < VEC; ++i)
                h[i] *= g[i];
        }
    }
    if(has_res)
    {
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            h[i] = fmaf(prm.res_scale, res[i], h[i]);
    }
}
template <int VEC, typename Get>
__device__ __forceinline__ void affine(const NormParams& prm, Get&& get, size_t at_w, size_t at_b, float mean, float rstd, float (&y)[VEC])
{
#pragma unroll
    for(int i = 0; i < VEC; ++i)
        y[i] = (y[i] - mean) * rstd;
    float p[VEC];
    if(prm.weight.ptr != nullptr)
    {
        get(prm.weight, at_w, p);
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            y[i] *= prm.weight_offset + p[i];
    }
    if(prm.bias.ptr != nullptr)
    {
        get(prm.bias, at_b, p);
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            y[i] += p[i];
    }
}

// The row stays in registers: every thread holds CNT groups of eight elements, group j * threads + t.  blockDim = (threads of a row,
// rows); more than one row per CTA only with at most a warp a row.  Bound by HBM for many rows (x, residual in, h, y out), by the chain load -
// sum - load - store for one.  SHIFT: rows and parameters start on any element's address; the groups then begin on y's 16-byte
// boundaries, the first and the last hold only some of the row, and the operands are shifted into place (one element at a time instead:
// 6 x 3075 30 us against 3.5, 1142 x 5287 fp32 with a bf16 residual 146 against 23, 4096 x 9001 952 against 126).
template <int CNT, bool X32, bool R32, bool SHIFT>
__global__ void __launch_bounds__(CNT == 1 || SHIFT ? 1024 : 512) norm_rows_kernel(const __grid_constant__ NormParams prm)
{
    __shared__ float red[4][32];
    const unsigned t = threadIdx.x, T = blockDim.x;
    const unsigned mine = blockIdx.x * blockDim.y + threadIdx.y, row = min(mine, prm.M - 1);
    const bool live     = mine < prm.M;
    grid_dependency_wait();
    grid_launch_dependents();
    if(!live && T >= 32)
        return; // (whole warps; where rows share a warp, all of its lanes take part in the sums)
    const int n = static_cast<int>(prm.n);
    const long long x_at = static_cast<long long>(row) * prm.x.ld, r_at = static_cast<long long>(row) * prm.res.ld;
    const long long h_at = static_cast<long long>(row) * prm.h.ld, y_at = static_cast<long long>(row) * prm.y.ld;
    // elements in front of the row in its first group
    const int before = SHIFT ? static_cast<int>((reinterpret_cast<uintptr_t>(prm.y.ptr) / (prm.y.dt == OUT_F32 ? 4 : 2) + y_at) & 7) : 0;
    auto first = [&](int j) { return static_cast<int>(j * T + t) * 8 - before; };        // column of a group's first element
    auto lo    = [&](int j) { return SHIFT ? max(0, -first(j)) : 0; };                   // the elements of the group that are the row's
    auto hi    = [&](int j) { return SHIFT ? min(8, n - first(j)) : 8; };
    auto some  = [&](int j) { return live && first(j) < n; };
    auto inside = [&](int j, int i) { return !SHIFT || (i >= lo(j) && i < hi(j)); };
    Raw<8, X32> rx[CNT];
    Raw<8, R32> rr[CNT];
    Pieces<X32> px[CNT];
    Pieces<R32> pr[CNT];
    const bool has_res   = prm.res.ptr != nullptr;
    const uint8_t* x_row = static_cast<const uint8_t*>(prm.x.ptr) + (x_at - before) * (X32 ? 4 : 2);
    const uint8_t* r_row = static_cast<const uint8_t*>(prm.res.ptr) + (r_at - before) * (R32 ? 4 : 2);
    const int sx = SHIFT ? shift_of<X32>(x_row) : 0, sr = SHIFT ? shift_of<R32>(r_row) : 0;
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        if(some(j))
        {
            if(SHIFT)
            {
                ld_pieces<X32>(px[j], x_row + (j * T + t) * (X32 ? 32u : 16u), sx, lo(j), hi(j));
                if(has_res)
                    ld_pieces<R32>(pr[j], r_row + (j * T + t) * (R32 ? 32u : 16u), sr, lo(j), hi(j));
            }
            else
            {
                ld_raw<8, X32>(rx[j], prm.x.ptr, x_at + first(j));
                if(has_res)
                    ld_raw<8, R32>(rr[j], prm.res.ptr, r_at + first(j));
            }
        }
    }
    float h[CNT][8];
    // values outside the row count for nothing in the sums
    auto clear_outside = [&](int j) {
        if(SHIFT && hi(j) - lo(j) != 8)
#pragma unroll
            for(int i = 0; i < 8; ++i)
                h[j][i] = inside(j, i) ? h[j][i] : 0.f;
    };
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        if(some(j))
        {
            if(SHIFT)
                align_pieces<X32>(rx[j], px[j], sx);
            unpack<8, X32>(rx[j], prm.x.dt, h[j]);
            clear_outside(j);
        }
        else
#pragma unroll
            for(int i = 0; i < 8; ++i)
                h[j][i] = 0.f;
    }
    auto stats = [&](int slot, float& mean, float& rstd) {
        mean = 0.f;
        if(prm.layer)
        {
            float s = 0.f;
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    s += h[j][i];
            mean = row_sum(s, red, slot) * prm.inv_n;
        }
        float s = 0.f;
#pragma unroll
        for(int j = 0; j < CNT; ++j)
            if(some(j))
            {
                float d[8];
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    d[i] = h[j][i] - mean;
                if(SHIFT && hi(j) - lo(j) != 8)
#pragma unroll
                    for(int i = 0; i < 8; ++i)
                        d[i] = inside(j, i) ? d[i] : 0.f;
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    s = fmaf(d[i], d[i], s);
            }
        rstd = rsqrtf(row_sum(s, red, slot + 1) * prm.inv_n + prm.eps);
    };
    float mean = 0.f, rstd = 1.f;
    if(prm.post)
        stats(0, mean, rstd);
    const size_t at_pw = param_at(prm.post_weight, row), at_pb = param_at(prm.post_bias, row), at_g = param_at(prm.gate, row);
    float gate1 = 1.f;
    if(prm.gate.ptr != nullptr && prm.gate_scalar)
    {
        float g[1];
        ld_param<1>(prm.gate.ptr, prm.gate.dt, at_g, g);
        gate1 = g[0];
    }
    auto getter = [&](int j) {
        return [&, j](const RowParam& q, size_t at, float (&v)[8]) {
            if(SHIFT)
                ld_param_shifted(q.ptr, q.dt, static_cast<long long>(at) + first(j), lo(j), hi(j), v);
            else
                ld_param<8>(q.ptr, q.dt, at + first(j), v);
        };
    };
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        if(some(j))
        {
            float r[8];
            if(has_res)
            {
                if(SHIFT)
                    align_pieces<R32>(rr[j], pr[j], sr);
                unpack<8, R32>(rr[j], prm.res.dt, r);
            }
            residual_sum<8>(prm, getter(j), at_pw, at_pb, at_g, gate1, mean, rstd, has_res, r, h[j]);
            clear_outside(j);
            if(prm.h.ptr != nullptr)
            {
                if(SHIFT)
                    st_shifted(prm.h.ptr, prm.h.dt, h_at + first(j), lo(j), hi(j), h[j]);
                else
                    st_vec<8>(prm.h.ptr, prm.h.dt, h_at + first(j), h[j]);
            }
        }
    }
    stats(2, mean, rstd);
    const size_t at_w = param_at(prm.weight, row), at_b = param_at(prm.bias, row);
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        if(some(j))
            affine<8>(prm, getter(j), at_w, at_b, mean, rstd, h[j]);
        if(SHIFT)
        {
            if(some(j))
                st_shifted(prm.y.ptr, prm.y.dt, y_at + first(j), lo(j), hi(j), h[j]);
        }
        else
            emit<8>(prm, row, first(j), some(j), h[j]);
    }
    if(!SHIFT && prm.y.dt >= OUT_E2M1)
        fill_scale_padding(prm.sf, row, prm.M, prm.n >> 5, t, T);
}

// A sum of any number of terms (Kahan, "Further remarks on reducing truncation errors", 1965): what an addition rounds off is carried
// to the next one, so the error stays at 2^-23 of the sum of magnitudes however many terms there are.
struct LongSum
{
    float sum = 0.f, lost = 0.f;
    __device__ __forceinline__ void add(float v)
    {
        const float y = v - lost, t = sum + y, off = (t - sum) - y;
        lost          = fabsf(off) <= 3.402823466e38f ? off : 0.f; // (an infinite sum stays one)
        sum           = t;
    }
};
// the values of a vector, added pairwise
template <int VEC>
__device__ __forceinline__ float pair_sum(const float (&v)[VEC])
{
    if(VEC == 1)
        return v[0];
    const int e = VEC == 1 ? 0 : 1;
    return ((v[0] + v[e]) + (v[2 * e] + v[3 * e])) + ((v[4 * e] + v[5 * e]) + (v[6 * e] + v[7 * e]));
}

// Rows that do not fit the registers: a CTA goes over its row once per sum and once for the outputs, recomputing h each
// time (the row comes from L2 after the first pass: 512 x 32768 56 us, of which 21 are its bytes at HBM's rate; rows on odd addresses
// go one element at a time, 300 x 32001 118 us).
template <int VEC>
__global__ void __launch_bounds__(512) norm_long_kernel(const __grid_constant__ NormParams prm)
{
    __shared__ float red[4][32];
    const unsigned t = threadIdx.x, T = blockDim.x, n = prm.n;
    const unsigned row = blockIdx.x;
    grid_dependency_wait();
    grid_launch_dependents();
    const bool has_res = prm.res.ptr != nullptr;
    const size_t at_pw = param_at(prm.post_weight, row), at_pb = param_at(prm.post_bias, row), at_g = param_at(prm.gate, row);
    const size_t at_w = param_at(prm.weight, row), at_b = param_at(prm.bias, row);
    float gate1 = 1.f;
    if(prm.gate.ptr != nullptr && prm.gate_scalar)
    {
        float g[1];
        ld_param<1>(prm.gate.ptr, prm.gate.dt, at_g, g);
        gate1 = g[0];
    }
    float pmean = 0.f, prstd = 1.f;
    auto load_x = [&](unsigned col, float (&v)[VEC]) {
        if(prm.x.dt == OUT_F32)
        {
            Raw<VEC, true> r;
            ld_raw<VEC, true>(r, prm.x.ptr, static_cast<size_t>(row) * prm.x.ld + col);
            unpack<VEC, true>(r, prm.x.dt, v);
        }
        else
        {
            Raw<VEC, false> r;
            ld_raw<VEC, false>(r, prm.x.ptr, static_cast<size_t>(row) * prm.x.ld + col);
            unpack<VEC, false>(r, prm.x.dt, v);
        }
    };
    auto load_h = [&](unsigned col, float (&v)[VEC]) {
        load_x(col, v);
        float r[VEC];
        if(has_res)
        {
            if(prm.res.dt == OUT_F32)
            {
                Raw<VEC, true> rr;
                ld_raw<VEC, true>(rr, prm.res.ptr, static_cast<size_t>(row) * prm.res.ld + col);
                unpack<VEC, true>(rr, prm.res.dt, r);
            }
            else
            {
                Raw<VEC, false> rr;
                ld_raw<VEC, false>(rr, prm.res.ptr, static_cast<size_t>(row) * prm.res.ld + col);
                unpack<VEC, false>(rr, prm.res.dt, r);
            }
        }
        auto get = [&](const RowParam& q, size_t at, float (&v)[VEC]) { ld_param<VEC>(q.ptr, q.dt, at + col, v); };
        residual_sum<VEC>(prm, get, at_pw, at_pb, at_g, gate1, pmean, prstd, has_res, r, v);
    };
    auto stats = [&](int slot, auto&& load, float& mean, float& rstd) {
        float m = 0.f;
        if(prm.layer)
        {
            LongSum s;
            for(unsigned col = t * VEC; col < n; col += T * VEC)
            {
                float v[VEC];
                load(col, v);
                s.add(pair_sum(v));
            }
            m = row_sum(s.sum, red, slot) * prm.inv_n;
        }
        LongSum s;
        for(unsigned col = t * VEC; col < n; col += T * VEC)
        {
            float v[VEC];
            load(col, v);
#pragma unroll
            for(int i = 0; i < VEC; ++i)
                v[i] = (v[i] - m) * (v[i] - m);
            s.add(pair_sum(v));
        }
        const float q = row_sum(s.sum, red, slot + 1) * prm.inv_n;
        mean          = m;
        rstd          = rsqrtf(q + prm.eps);
    };
    if(prm.post)
        stats(0, load_x, pmean, prstd);
    float mean, rstd;
    stats(2, load_h, mean, rstd);
    // (whole warps go round together: the block scales are shared by shuffles)
    for(unsigned c0 = 0; c0 < n; c0 += T * VEC)
    {
        const unsigned col = c0 + t * VEC;
        const bool in      = col < n;
        float v[VEC];
#pragma unroll
        for(int i = 0; i < VEC; ++i)
            v[i] = 0.f;
        if(in)
        {
            load_h(col, v);
            if(prm.h.ptr != nullptr)
                st_vec<VEC>(prm.h.ptr, prm.h.dt, static_cast<size_t>(row) * prm.h.ld + col, v);
            auto get = [&](const RowParam& q, size_t at, float (&v)[VEC]) { ld_param<VEC>(q.ptr, q.dt, at + col, v); };
            affine<VEC>(prm, get, at_w, at_b, mean, rstd, v);
        }
        emit<VEC>(prm, row, col, in, v);
    }
    if(prm.y.dt >= OUT_E2M1)
        fill_scale_padding(prm.sf, row, prm.M, n >> 5, t, T);
}

// ------------------------------------------------------------------------------------------- gated activation
struct ActMulParams
{
    const void* in;
    long long in_ld; // elements between rows; a row is [n gate values][n factors]
    void* out;
    long long out_ld;
    int in_dt, out_dt, act;
    unsigned M, n;
    unsigned row_vecs; // vectors of eight per row, the partial ones included (plain outputs)
    BlockScales sf;
};

// Plain outputs: a thread takes U vectors of eight, 256 vectors apart, of the flat list of all rows' vectors; HBM-bound
// (16384 x 12288: relu 173 us, silu 177, gelu_tanh 180, 6.7 to 7.0 TB/s; gelu 205, whose arithmetic shows).  Compiled per activation: with all of them in
// one kernel 190 and 207 us.
template <bool X32, int ACT>
__global__ void __launch_bounds__(256) act_mul_kernel(const __grid_constant__ ActMulParams prm)
{
    constexpr int U = 2;
    grid_dependency_wait();
    grid_launch_dependents();
    const unsigned long long total = static_cast<unsigned long long>(prm.M) * prm.row_vecs;
    const unsigned long long first = static_cast<unsigned long long>(blockIdx.x) * (256 * U) + threadIdx.x;
    Raw<8, X32> a[U], b[U];
    size_t out_at[U];
#pragma unroll
    for(int u = 0; u < U; ++u)
    {
        const unsigned long long i = first + static_cast<unsigned long long>(u) * 256;
        if(i < total)
        {
            const unsigned row = total <= 0xFFFFFFFFull ? static_cast<unsigned>(i) / prm.row_vecs : static_cast<unsigned>(i / prm.row_vecs);
            const unsigned col = static_cast<unsigned>(i - static_cast<unsigned long long>(row) * prm.row_vecs) * 8;
            const size_t at    = static_cast<size_t>(row) * prm.in_ld + col;
            ld_raw<8, X32>(a[u], prm.in, at);
            ld_raw<8, X32>(b[u], prm.in, at + prm.n);
            out_at[u] = static_cast<size_t>(row) * prm.out_ld + col;
        }
    }
#pragma unroll
    for(int u = 0; u < U; ++u)
    {
        if(first + static_cast<unsigned long long>(u) * 256 < total)
        {
            float g[8], v[8];
            unpack<8, X32>(a[u], prm.in_dt, g);
            unpack<8, X32>(b[u], prm.in_dt, v);
            activate<ACT>(g, prm.act);
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] *= g[i];
            st_vec<8>(prm.out, prm.out_dt, out_at[u], v);
        }
    }
}

// Rows that start on any element's address: a thread's eight outputs begin on a 16-byte boundary of the output's row (its first and
// last groups are partial), their operands are shifted into place (8192 x 1001 15.8 us, one element at a time 26).
template <bool X32, int ACT>
__global__ void __launch_bounds__(256) act_mul_shift_kernel(const __grid_constant__ ActMulParams prm)
{
    constexpr int U = X32 ? 1 : 2;
    grid_dependency_wait();
    grid_launch_dependents();
    const unsigned long long total = static_cast<unsigned long long>(prm.M) * prm.row_vecs;
    const unsigned long long first = static_cast<unsigned long long>(blockIdx.x) * (256 * U) + threadIdx.x;
    const int in_size = X32 ? 4 : 2, out_size = prm.out_dt == OUT_F32 ? 4 : 2;
    Pieces<X32> a[U], b[U];
    int sa[U], sb[U], lo[U], hi[U];
    long long out_at[U];
#pragma unroll
    for(int u = 0; u < U; ++u)
    {
        const unsigned long long i = first + static_cast<unsigned long long>(u) * 256;
        lo[u] = hi[u] = 0;
        if(i < total)
        {
            const unsigned row   = total <= 0xFFFFFFFFull ? static_cast<unsigned>(i) / prm.row_vecs : static_cast<unsigned>(i / prm.row_vecs);
            const unsigned group = static_cast<unsigned>(i - static_cast<unsigned long long>(row) * prm.row_vecs);
            const long long dst  = static_cast<long long>(row) * prm.out_ld;
            const int before     = static_cast<int>((reinterpret_cast<uintptr_t>(prm.out) + dst * out_size) & 15) / out_size; // elements of the first group in front of the row
            const long long col  = static_cast<long long>(group) * 8 - before;
            lo[u]                = group == 0 ? before : 0;
            hi[u]                = static_cast<int>(min(8ll, static_cast<long long>(prm.n) - col));
            out_at[u]            = dst + col;
            if(lo[u] < hi[u])
            {
                const uint8_t* src = static_cast<const uint8_t*>(prm.in) + (static_cast<long long>(row) * prm.in_ld + col) * in_size;
                const uint8_t* factor = src + static_cast<size_t>(prm.n) * in_size;
                sa[u] = shift_of<X32>(src), sb[u] = shift_of<X32>(factor);
                ld_pieces<X32>(a[u], src, sa[u], lo[u], hi[u]);
                ld_pieces<X32>(b[u], factor, sb[u], lo[u], hi[u]);
            }
        }
    }
#pragma unroll
    for(int u = 0; u < U; ++u)
    {
        if(lo[u] < hi[u])
        {
            float g[8], v[8];
            Raw<8, X32> r;
            align_pieces<X32>(r, a[u], sa[u]);
            unpack<8, X32>(r, prm.in_dt, g);
            align_pieces<X32>(r, b[u], sb[u]);
            unpack<8, X32>(r, prm.in_dt, v);
            activate<ACT>(g, prm.act);
#pragma unroll
            for(int i = 0; i < 8; ++i)
                v[i] *= g[i];
            if(hi[u] - lo[u] == 8)
                st_vec<8>(static_cast<uint8_t*>(prm.out) + out_at[u] * out_size, prm.out_dt, 0, v);
            else
            {
#pragma unroll
                for(int i = 0; i < 8; ++i)
                    if(i >= lo[u] && i < hi[u])
                        store_out(static_cast<uint8_t*>(prm.out) + (out_at[u] + i) * out_size, 0, v[i], prm.out_dt);
            }
        }
    }
}

// MX outputs: a CTA of eight warps takes 32 rows x 8 blocks (256 columns), four rows a warp, so that the tile's 256 scale
// bytes, one chunk of either GEMM layout, are collected in shared memory and leave in whole words.
template <bool X32, bool FP4, int ACT>
__global__ void __launch_bounds__(256) act_mul_mx_kernel(const __grid_constant__ ActMulParams prm)
{
    __shared__ __align__(16) uint8_t sf_tile[256];
    grid_dependency_wait();
    grid_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned kblocks = prm.n >> 5, k_tiles = (kblocks + 7) / 8;
    const unsigned tm = blockIdx.x / k_tiles, tk = blockIdx.x - tm * k_tiles;
    const unsigned col = tk * 256 + lane * 8;
    const bool col_in  = col < prm.n;
    Raw<8, X32> a[4], b[4];
#pragma unroll
    for(int u = 0; u < 4; ++u)
    {
        const unsigned row = tm * 32 + warp * 4 + u;
        if(col_in && row < prm.M)
        {
            const size_t at = static_cast<size_t>(row) * prm.in_ld + col;
            ld_raw<8, X32>(a[u], prm.in, at);
            ld_raw<8, X32>(b[u], prm.in, at + prm.n);
        }
    }
#pragma unroll
    for(int u = 0; u < 4; ++u)
    {
        const unsigned r = warp * 4 + u, row = tm * 32 + r;
        const bool ok = col_in && row < prm.M;
        float g[8], v[8];
        if(ok)
        {
            unpack<8, X32>(a[u], prm.in_dt, g);
            unpack<8, X32>(b[u], prm.in_dt, v);
            activate<ACT>(g, prm.act);
        }
#pragma unroll
        for(int i = 0; i < 8; ++i)
            v[i] = ok ? v[i] * g[i] : 0.f;
        uint32_t q[2];
        uint32_t byte = mx_block<FP4>(v, q);
        if(ok)
        {
            uint8_t* dst = static_cast<uint8_t*>(prm.out) + static_cast<size_t>(row) * prm.out_ld;
            if(FP4)
                *reinterpret_cast<uint32_t*>(dst + (col >> 1)) = q[0];
            else
                *reinterpret_cast<uint2*>(dst + col) = make_uint2(q[0], q[1]);
        }
        else
            byte = prm.sf.layout == QSL_M32K4 ? 0x7F : 0;
        if((lane & 3) == 0)
        {
            const int kb = lane >> 2;
            int pos      = r * 8 + kb;
            if(prm.sf.layout == QSL_E8M0_SHUFFLE)
                pos = (kb & 3) * 64 + (r & 15) * 4 + (kb >> 2) * 2 + (r >> 4);
            else if(prm.sf.layout == QSL_M32K4)
                pos = (kb >> 2) * 128 + r * 4 + (kb & 3);
            sf_tile[pos] = static_cast<uint8_t>(byte);
        }
    }
    __syncthreads();
    if(prm.sf.layout == QSL_PLAIN)
    {
        // 8 bytes per row, one a thread
        const unsigned row = tm * 32 + (threadIdx.x >> 3), kb = tk * 8 + (threadIdx.x & 7);
        if(row < prm.M && kb < kblocks)
            prm.sf.ptr[static_cast<size_t>(row) * prm.sf.cols + kb] = sf_tile[threadIdx.x];
    }
    else if(threadIdx.x < 64)
    {
        // (m/32,k/4,32,4): the second half of the chunk only if the array has it
        uint8_t* dst = prm.sf.ptr + static_cast<size_t>(tm) * (static_cast<size_t>(prm.sf.cols) * 32) + tk * 256;
        if(prm.sf.layout == QSL_E8M0_SHUFFLE || tk * 8 + (threadIdx.x >> 5) * 4 < kblocks)
            reinterpret_cast<uint32_t*>(dst)[threadIdx.x] = reinterpret_cast<const uint32_t*>(sf_tile)[threadIdx.x];
    }
}

} // namespace b200
