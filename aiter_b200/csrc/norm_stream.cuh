// gated_residual_norm for many rows: persistent CTAs that stream their rows through shared memory.
//
// The operator moves x and the residual in and h and y out, 8 bytes an element in 16-bit types, and is bound by HBM as long as
// an SM always has some 50 KB of loads under way and spends less than about 25 instructions an element.  Hence: a CTA owns a
// contiguous block of rows and keeps the next ones in flight with bulk copies (one thread, two instructions a row, no
// registers), while the current row goes from shared memory to registers, through its one or two norms and out; a thread holds
// 16 to 32 values, over which the fixed work of a row (two sums, addresses) is spread; types are compile-time and the arithmetic
// is two values an instruction.
//
// Rows that start on any address are copied from the 16-byte boundary below to the one above, and read pair by pair.
#pragma once
#include "block_ops.cuh"

namespace b200 {

struct NormStreamLayout
{
    unsigned x_bytes, r_bytes; // shared memory of one row, multiples of 16
    unsigned stages;
    unsigned param_off;        // unaligned rows: where the parameters of the current entry are kept as fp32, pitch param_pitch floats
    unsigned param_pitch;
    WaitReport report;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__host__ __device__ constexpr int esize_of(int dt) { return dt == OUT_F32 ? 4 : 2; }
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w)
{
    if(DT == OUT_BF16)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// VEC consecutive elements of a compile-time type as pairs.  VEC = 8: aligned to the vector.  VEC = 2: aligned to the element
// only (`even`: to the pair), and the second element exists only if `two`.
template <int DT, int VEC>
__device__ __forceinline__ void rd_vec(const uint8_t* p, bool even, bool two, float2 (&v)[VEC / 2])
{
    if constexpr(VEC == 2)
    {
        if constexpr(DT == OUT_F32)
        {
            if(even && two)
                v[0] = *reinterpret_cast<const float2*>(p);
            else
                v[0] = make_float2(reinterpret_cast<const float*>(p)[0], two ? reinterpret_cast<const float*>(p)[1] : 0.f);
        }
        else
        {
            uint32_t w;
            if(even && two)
                w = *reinterpret_cast<const uint32_t*>(p);
            else
                w = reinterpret_cast<const uint16_t*>(p)[0] | (two ? static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[1]) << 16 : 0u);
            v[0] = unpack2<DT>(w);
        }
    }
    else if constexpr(DT == OUT_F32)
    {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
    }
    else
    {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        v[0] = unpack2<DT>(a.x), v[1] = unpack2<DT>(a.y), v[2] = unpack2<DT>(a.z), v[3] = unpack2<DT>(a.w);
    }
}
template <int DT, int VEC>
__device__ __forceinline__ void wr_vec(uint8_t* p, bool even, bool two, const float2 (&v)[VEC / 2])
{
    if constexpr(VEC == 2)
    {
        if constexpr(DT == OUT_F32)
        {
            if(even && two)
                *reinterpret_cast<float2*>(p) = v[0];
            else
            {
                reinterpret_cast<float*>(p)[0] = v[0].x;
                if(two)
                    reinterpret_cast<float*>(p)[1] = v[0].y;
            }
        }
        else
        {
            const uint32_t w = pack_out16x2(v[0].x, v[0].y, DT == OUT_F16);
            if(even && two)
                *reinterpret_cast<uint32_t*>(p) = w;
            else
            {
                reinterpret_cast<uint16_t*>(p)[0] = static_cast<uint16_t>(w);
                if(two)
                    reinterpret_cast<uint16_t*>(p)[1] = static_cast<uint16_t>(w >> 16);
            }
        }
    }
    else if constexpr(DT == OUT_F32)
    {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
    else
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_out16x2(v[0].x, v[0].y, DT == OUT_F16), pack_out16x2(v[1].x, v[1].y, DT == OUT_F16),
                                                  pack_out16x2(v[2].x, v[2].y, DT == OUT_F16), pack_out16x2(v[3].x, v[3].y, DT == OUT_F16));
}
// every pair of a row starts on a boundary of its size
template <int DT>
__device__ __forceinline__ bool pairs_aligned(const void* p)
{
    return (reinterpret_cast<uintptr_t>(p) & (2 * esize_of(DT) - 1)) == 0;
}

// h *= offset + p  and  h += p for a parameter vector p of the row
template <int PD, int VEC, int CNT>
__device__ __forceinline__ void scale_by(float2 (&h)[CNT][VEC / 2], const uint8_t* p, unsigned col0, unsigned col_step, unsigned n, float offset)
{
    const bool even = pairs_aligned<PD>(p);
    const float2 o  = make_float2(offset, offset);
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        const unsigned col = col0 + j * col_step;
        if(col < n)
        {
            float2 q[VEC / 2];
            rd_vec<PD, VEC>(p + col * esize_of(PD), even, col + 1 < n, q);
#pragma unroll
            for(int k = 0; k < VEC / 2; ++k)
                h[j][k] = __fmul2_rn(h[j][k], __fadd2_rn(q[k], o));
        }
    }
}
template <int PD, int VEC, int CNT>
__device__ __forceinline__ void shift_by(float2 (&h)[CNT][VEC / 2], const uint8_t* p, unsigned col0, unsigned col_step, unsigned n)
{
    const bool even = pairs_aligned<PD>(p);
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        const unsigned col = col0 + j * col_step;
        if(col < n)
        {
            float2 q[VEC / 2];
            rd_vec<PD, VEC>(p + col * esize_of(PD), even, col + 1 < n, q);
#pragma unroll
            for(int k = 0; k < VEC / 2; ++k)
                h[j][k] = __fadd2_rn(h[j][k], q[k]);
        }
    }
}
// the row's vectors as an MX operand
template <bool FP4, int CNT>
__device__ __forceinline__ void emit_mx(const BlockScales& sf, uint8_t* y, unsigned row, unsigned col0, unsigned col_step, unsigned n, const float2 (&h)[CNT][4])
{
    uint8_t* const sf_row = sf.ptr + sf_offset(sf, row, 0); // (block 0; the others lie at offsets that do not depend on the row)
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        const unsigned col = col0 + j * col_step;
        const bool in      = col < n;
        const float f[8]   = {h[j][0].x, h[j][0].y, h[j][1].x, h[j][1].y, h[j][2].x, h[j][2].y, h[j][3].x, h[j][3].y};
        uint32_t q[2];
        uint32_t byte = mx_block<FP4>(f, q);
        if(in)
        {
            if(FP4)
                *reinterpret_cast<uint32_t*>(y + (col >> 1)) = q[0];
            else
                *reinterpret_cast<uint2*>(y + col) = make_uint2(q[0], q[1]);
        }
        const unsigned kb = col >> 5;
        if(sf.layout == QSL_M32K4)
        {
            // four neighbouring blocks of a row are four neighbouring bytes: one word per 16 lanes
            byte |= __shfl_down_sync(0xffffffffu, byte, 4) << 8;
            byte |= __shfl_down_sync(0xffffffffu, byte, 8) << 16;
            if(in && (threadIdx.x & 15) == 0)
                *reinterpret_cast<uint32_t*>(sf_row + (kb >> 2) * 128u) = byte;
        }
        else if(in && (threadIdx.x & 3) == 0)
            sf_row[sf.layout == QSL_E8M0_SHUFFLE ? (kb >> 3) * 256u + (kb & 3) * 64u + ((kb >> 2) & 1) * 2u : kb] = static_cast<uint8_t>(byte);
    }
}

// XD, RD: types of x and of the residual and h; PD: of every parameter of more than one value.  A thread holds CNT vectors of VEC
// elements, vector j at element (j * threads + t) * VEC.
template <int XD, int RD, int PD, int VEC, int CNT>
__global__ void __launch_bounds__(512, VEC * CNT <= 16 ? 2 : 1) norm_stream_kernel(const __grid_constant__ NormParams prm, const __grid_constant__ NormStreamLayout lay)
{
    constexpr int P = VEC / 2;
    constexpr int XS = esize_of(XD), RS = esize_of(RD), PS = esize_of(PD);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float red[8][32]; // two sets of slots, for even and odd rows: one barrier a sum is enough
    __shared__ __align__(8) uint64_t full[4];
    const unsigned t = threadIdx.x, T = blockDim.x, n = prm.n;
    const bool has_res = prm.res.ptr != nullptr, has_h = prm.h.ptr != nullptr, has_w = prm.weight.ptr != nullptr, has_b = prm.bias.ptr != nullptr;
    const bool post = prm.post != 0, has_pw = prm.post_weight.ptr != nullptr, has_pb = prm.post_bias.ptr != nullptr;
    const bool gate_vec = prm.gate.ptr != nullptr && !prm.gate_scalar, gate_one = prm.gate.ptr != nullptr && prm.gate_scalar;
    // this CTA's rows: the first `extra` CTAs take one more
    const unsigned per = prm.M / gridDim.x, extra = prm.M % gridDim.x;
    const unsigned row0 = blockIdx.x * per + min(blockIdx.x, extra);
    const unsigned rows = per + (blockIdx.x < extra ? 1u : 0u);
    const unsigned S = lay.stages, stage_bytes = lay.x_bytes + lay.r_bytes;
    if(t == 0)
    {
        for(unsigned s = 0; s < S; ++s)
            mbar_init(smem_u32(&full[s]), 1);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    const uint8_t* xg = static_cast<const uint8_t*>(prm.x.ptr) + static_cast<size_t>(row0) * prm.x.ld * XS;
    const uint8_t* rg = static_cast<const uint8_t*>(prm.res.ptr) + static_cast<size_t>(row0) * prm.res.ld * RS;
    auto load = [&](const uint8_t* xp, const uint8_t* rp, unsigned s) { // a row into stage s, by one thread
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem) + s * stage_bytes;
        const unsigned xo  = VEC == 8 ? 0u : static_cast<unsigned>(reinterpret_cast<uintptr_t>(xp) & 15);
        const unsigned ro  = VEC == 8 ? 0u : static_cast<unsigned>(reinterpret_cast<uintptr_t>(rp) & 15);
        const unsigned xb  = (xo + n * XS + 15u) & ~15u;
        const unsigned rb  = has_res ? (ro + n * RS + 15u) & ~15u : 0u;
        mbar_arrive_expect_tx(bar, xb + rb);
        bulk_load(dst, xp - xo, xb, bar);
        if(has_res)
            bulk_load(dst + lay.x_bytes, rp - ro, rb, bar);
    };
    const size_t x_step = static_cast<size_t>(prm.x.ld) * XS, r_step = static_cast<size_t>(prm.res.ld) * RS;
    if(t == 0)
        for(unsigned i = 0; i < min(S, rows); ++i)
            load(xg + i * x_step, rg + i * r_step, i);
    const unsigned y_size = bytes_of_mode(prm.y.dt);
    uint8_t* hg = static_cast<uint8_t*>(prm.h.ptr) + static_cast<size_t>(row0) * prm.h.ld * RS;
    uint8_t* yg = static_cast<uint8_t*>(prm.y.ptr) + static_cast<size_t>(row0) * prm.y.ld * y_size;
    const size_t h_step = static_cast<size_t>(prm.h.ld) * RS, y_step = static_cast<size_t>(prm.y.ld) * y_size;
    // The parameters' entries of the current row, until row `change`.  With unaligned rows they are kept in shared memory as fp32
    // (an entry of an odd number of 16-bit values is as unaligned as the rows, and every row of the CTA reads it again).
    constexpr int QD = VEC == 2 ? OUT_F32 : PD;
    const uint8_t *w = nullptr, *b = nullptr, *pw = nullptr, *pb = nullptr, *pg = nullptr;
    float gate1     = 1.f;
    unsigned change = 0xFFFFFFFFu;
    auto entries    = [&](unsigned row) {
        int k     = 0;
        auto take = [&](const RowParam& q, const uint8_t*& at) {
            const uint8_t* src = static_cast<const uint8_t*>(q.ptr) + param_at(q, row) * PS;
            if(q.ld != 0)
                change = min(change, (row / q.rows_per + 1) * q.rows_per);
            at = src;
            if(VEC == 2 && q.ptr != nullptr)
            {
                float* dst = reinterpret_cast<float*>(smem + lay.param_off) + (k++) * lay.param_pitch;
                for(unsigned e = t; e < n; e += T)
                    dst[e] = load_elem_any(src, PD, e);
                at = reinterpret_cast<const uint8_t*>(dst);
            }
        };
        change = 0xFFFFFFFFu;
        if(VEC == 2)
            __syncthreads(); // nobody reads the previous entries any more
        take(prm.weight, w);
        take(prm.bias, b);
        take(prm.post_weight, pw);
        take(prm.post_bias, pb);
        if(gate_vec)
            take(prm.gate, pg);
        else if(gate_one)
        {
            if(prm.gate.ld != 0)
                change = min(change, (row / prm.gate.rows_per + 1) * prm.gate.rows_per);
            gate1 = load_elem_any(prm.gate.ptr, prm.gate.dt, param_at(prm.gate, row));
        }
        if(VEC == 2)
            __syncthreads();
    };
    entries(row0);
    unsigned s = 0, phase = 0;
    bool expired = false;
    const unsigned col0 = t * VEC, col_step = T * VEC;
#pragma unroll 1
    for(unsigned i = 0; i < rows; ++i)
    {
        if(row0 + i >= change) // (the same for every thread)
            entries(row0 + i);
        // (bounded, though a copy of valid memory always completes: on expiry the status record says that the output is incomplete)
        if(!expired && !mbar_try_wait(smem_u32(&full[s]), phase))
        {
            const uint64_t t0 = global_timer_ns();
            while(!expired && !mbar_try_wait_parked(smem_u32(&full[s]), phase, kParkNs))
                expired = global_timer_ns() - t0 > kWaitLimitNs;
            if(expired)
                report_timeout(lay.report, ST_TIMEOUT_ROWS, i);
        }
        const uint8_t* xs = smem + s * stage_bytes;
        const uint8_t* rs = xs + lay.x_bytes;
        if(VEC != 8)
        {
            xs += reinterpret_cast<uintptr_t>(xg) & 15;
            rs += reinterpret_cast<uintptr_t>(rg) & 15;
        }
        float2 h[CNT][P];
        {
            const bool even = pairs_aligned<XD>(xs);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(col < n)
                    rd_vec<XD, VEC>(xs + col * XS, even, col + 1 < n, h[j]);
                else
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = make_float2(0.f, 0.f);
            }
        }
        auto stats = [&](int slot, float& mean, float& rstd) {
            slot += 4 * static_cast<int>(i & 1);
            float2 a = make_float2(0.f, 0.f);
            mean     = 0.f;
            if(prm.layer)
            {
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        a = __fadd2_rn(a, h[j][k]);
                mean = row_sum(a.x + a.y, red, slot) * prm.inv_n;
                a    = make_float2(0.f, 0.f);
                const float2 m = make_float2(-mean, -mean);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
                {
                    const unsigned col = col0 + j * col_step;
                    if(col < n)
#pragma unroll
                        for(int k = 0; k < P; ++k)
                        {
                            float2 d = __fadd2_rn(h[j][k], m);
                            if(VEC == 2 && col + 1 >= n)
                                d.y = 0.f;
                            a = __ffma2_rn(d, d, a);
                        }
                }
            }
            else
            {
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        a = __ffma2_rn(h[j][k], h[j][k], a);
            }
            rstd = rsqrtf(row_sum(a.x + a.y, red, slot + 1) * prm.inv_n + prm.eps);
        };
        float mean = 0.f, rstd = 1.f;
        if(post)
        {
            stats(0, mean, rstd);
            const float2 a = make_float2(rstd, rstd);
            if(prm.layer)
            {
                const float2 m = make_float2(-mean, -mean);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __fadd2_rn(h[j][k], m);
            }
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = __fmul2_rn(h[j][k], a);
            if(has_pw)
                scale_by<QD, VEC, CNT>(h, pw, col0, col_step, n, 0.f);
            if(has_pb)
                shift_by<QD, VEC, CNT>(h, pb, col0, col_step, n);
        }
        if(gate_vec)
            scale_by<QD, VEC, CNT>(h, pg, col0, col_step, n, 0.f);
        else if(gate_one)
        {
            const float2 a = make_float2(gate1, gate1);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = __fmul2_rn(h[j][k], a);
        }
        if(has_res)
        {
            const float2 a  = make_float2(prm.res_scale, prm.res_scale);
            const bool even = pairs_aligned<RD>(rs);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(col < n)
                {
                    float2 q[P];
                    rd_vec<RD, VEC>(rs + col * RS, even, col + 1 < n, q);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __ffma2_rn(a, q[k], h[j][k]);
                }
            }
        }
        // elements behind the row count for nothing in the sums (a first layer norm or its bias has touched them)
        if(post)
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(col >= n)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = make_float2(0.f, 0.f);
                else if(VEC == 2 && col + 1 >= n)
                    h[j][0].y = 0.f;
            }
        if(has_h)
        {
            const bool even = pairs_aligned<RD>(hg);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(col < n)
                    wr_vec<RD, VEC>(hg + col * RS, even, col + 1 < n, h[j]);
            }
        }
        stats(2, mean, rstd);
        // every thread has read its part of the stage (the sum's barrier): a later row may land there
        if(t == 0 && i + S < rows && !expired)
            load(xg + S * x_step, rg + S * r_step, s);
        if(++s == S)
        {
            s = 0;
            phase ^= 1u;
        }
        {
            const float2 a = make_float2(rstd, rstd);
            if(prm.layer)
            {
                const float2 m = make_float2(-mean, -mean);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __fadd2_rn(h[j][k], m);
            }
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = __fmul2_rn(h[j][k], a);
        }
        if(has_w)
            scale_by<QD, VEC, CNT>(h, w, col0, col_step, n, prm.weight_offset);
        if(has_b)
            shift_by<QD, VEC, CNT>(h, b, col0, col_step, n);
        // one test of y's type a row
        auto store_all = [&](auto tag) {
            constexpr int YD = decltype(tag)::value;
            const bool even  = pairs_aligned<YD>(yg);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(col < n)
                    wr_vec<YD, VEC>(yg + col * esize_of(YD), even, col + 1 < n, h[j]);
            }
        };
        if(prm.y.dt == OUT_BF16)
            store_all(std::integral_constant<int, OUT_BF16>{});
        else if(prm.y.dt == OUT_F16)
            store_all(std::integral_constant<int, OUT_F16>{});
        else if(prm.y.dt == OUT_F32)
            store_all(std::integral_constant<int, OUT_F32>{});
        else if constexpr(VEC == 8)
        {
            const unsigned row = row0 + i;
            if(prm.y.dt == OUT_E2M1)
                emit_mx<true, CNT>(prm.sf, yg, row, col0, col_step, n, h);
            else
                emit_mx<false, CNT>(prm.sf, yg, row, col0, col_step, n, h);
            if(prm.sf.layout != QSL_PLAIN && (row == prm.M - 1 || (n & 255) != 0))
                fill_scale_padding(prm.sf, row, prm.M, n >> 5, t, T);
        }
        xg += x_step;
        rg += r_step;
        hg += h_step;
        yg += y_step;
    }
    if(expired)
    {
        // copies still in flight land before this CTA's shared memory is released (bounded)
        const uint64_t t0 = global_timer_ns();
        while(global_timer_ns() - t0 < 200000ull) {}
    }
}

// Short rows (at most 256 values, as the norm of a head has them), many of them: LANES threads a row, 32 / LANES rows a warp and
// four such groups of rows a thread, whose loads are all under way before the first sum.
template <int XD, int RD, int PD, int LANES>
__global__ void __launch_bounds__(256) norm_short_kernel(const __grid_constant__ NormParams prm)
{
    constexpr int U = 4, R = 32 / LANES;
    constexpr int XS = esize_of(XD), RS = esize_of(RD), PS = esize_of(PD);
    grid_dependency_wait();
    grid_launch_dependents();
    const unsigned lane = threadIdx.x & 31, n = prm.n;
    const unsigned col = (lane % LANES) * 8;
    const bool col_in  = col < n;
    const size_t first = (static_cast<size_t>(blockIdx.x) * 8 + (threadIdx.x >> 5)) * (U * R) + lane / LANES;
    const bool has_res = prm.res.ptr != nullptr;
    Raw<8, XD == OUT_F32> rx[U];
    Raw<8, RD == OUT_F32> rr[U];
#pragma unroll
    for(int u = 0; u < U; ++u)
    {
        const size_t row = first + u * R;
        if(col_in && row < prm.M)
        {
            ld_raw<8, XD == OUT_F32>(rx[u], prm.x.ptr, row * prm.x.ld + col);
            if(has_res)
                ld_raw<8, RD == OUT_F32>(rr[u], prm.res.ptr, row * prm.res.ld + col);
        }
    }
    auto sum = [](float v) {
#pragma unroll
        for(int d = LANES / 2; d > 0; d >>= 1)
            v += __shfl_xor_sync(0xffffffffu, v, d);
        return v;
    };
#pragma unroll 1
    for(int u = 0; u < U; ++u)
    {
        // (the unrolled copies are selected by u: the raw registers stay registers)
        Raw<8, XD == OUT_F32> cx = rx[0];
        Raw<8, RD == OUT_F32> cr = rr[0];
#pragma unroll
        for(int k = 0; k + 1 < U; ++k)
        {
            rx[k] = rx[k + 1];
            rr[k] = rr[k + 1];
        }
        const size_t row_l = first + u * R;
        const bool in      = col_in && row_l < prm.M;
        const unsigned row = static_cast<unsigned>(row_l < prm.M ? row_l : 0);
        float v[8];
        if(in)
            unpack<8, XD == OUT_F32>(cx, XD, v);
        float2 h[1][4];
#pragma unroll
        for(int k = 0; k < 4; ++k)
            h[0][k] = in ? make_float2(v[2 * k], v[2 * k + 1]) : make_float2(0.f, 0.f);
        auto stats = [&](float& mean, float& rstd) {
            mean = 0.f;
            if(prm.layer)
                mean = sum(((h[0][0].x + h[0][0].y) + (h[0][1].x + h[0][1].y)) + ((h[0][2].x + h[0][2].y) + (h[0][3].x + h[0][3].y))) * prm.inv_n;
            float2 a       = make_float2(0.f, 0.f);
            const float2 m = make_float2(-mean, -mean);
            if(in)
#pragma unroll
                for(int k = 0; k < 4; ++k)
                {
                    const float2 d = __fadd2_rn(h[0][k], m);
                    a              = __ffma2_rn(d, d, a);
                }
            rstd = rsqrtf(sum(a.x + a.y) * prm.inv_n + prm.eps);
        };
        auto normalise = [&](float mean, float rstd) {
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[0][k] = __fmul2_rn(__fadd2_rn(h[0][k], make_float2(-mean, -mean)), make_float2(rstd, rstd));
        };
        auto entry = [&](const RowParam& q) { return static_cast<const uint8_t*>(q.ptr) + param_at(q, row) * PS; };
        float mean, rstd;
        if(prm.post)
        {
            stats(mean, rstd);
            normalise(mean, rstd);
            if(prm.post_weight.ptr != nullptr)
                scale_by<PD, 8, 1>(h, entry(prm.post_weight), col, 0, n, 0.f);
            if(prm.post_bias.ptr != nullptr)
                shift_by<PD, 8, 1>(h, entry(prm.post_bias), col, 0, n);
        }
        if(prm.gate.ptr != nullptr)
        {
            if(prm.gate_scalar)
            {
                const float g = load_elem_any(prm.gate.ptr, prm.gate.dt, param_at(prm.gate, row));
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    h[0][k] = __fmul2_rn(h[0][k], make_float2(g, g));
            }
            else
                scale_by<PD, 8, 1>(h, entry(prm.gate), col, 0, n, 0.f);
        }
        if(has_res && in)
        {
            unpack<8, RD == OUT_F32>(cr, RD, v);
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[0][k] = __ffma2_rn(make_float2(prm.res_scale, prm.res_scale), make_float2(v[2 * k], v[2 * k + 1]), h[0][k]);
        }
        if(!in)
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[0][k] = make_float2(0.f, 0.f);
        if(prm.h.ptr != nullptr && in)
            wr_vec<RD, 8>(static_cast<uint8_t*>(prm.h.ptr) + (static_cast<size_t>(row) * prm.h.ld + col) * RS, true, true, h[0]);
        stats(mean, rstd);
        normalise(mean, rstd);
        if(prm.weight.ptr != nullptr)
            scale_by<PD, 8, 1>(h, entry(prm.weight), col, 0, n, prm.weight_offset);
        if(prm.bias.ptr != nullptr)
            shift_by<PD, 8, 1>(h, entry(prm.bias), col, 0, n);
        uint8_t* y = static_cast<uint8_t*>(prm.y.ptr) + static_cast<size_t>(row) * prm.y.ld * bytes_of_mode(prm.y.dt);
        if(prm.y.dt >= OUT_E2M1)
        {
            // (a lane whose row or column does not exist takes part in the block's maximum with its neighbours, which do not either)
            const unsigned limit = in ? n : 0u;
            if(prm.y.dt == OUT_E2M1)
                emit_mx<true, 1>(prm.sf, y, row, col, 0, limit, h);
            else
                emit_mx<false, 1>(prm.sf, y, row, col, 0, limit, h);
            if(row_l < prm.M)
                fill_scale_padding(prm.sf, row, prm.M, n >> 5, lane % LANES, LANES);
        }
        else if(in)
        {
            if(prm.y.dt == OUT_BF16)
                wr_vec<OUT_BF16, 8>(y + col * 2, true, true, h[0]);
            else if(prm.y.dt == OUT_F16)
                wr_vec<OUT_F16, 8>(y + col * 2, true, true, h[0]);
            else
                wr_vec<OUT_F32, 8>(y + col * 4, true, true, h[0]);
        }
    }
}

} // namespace b200
