// gated_residual_norm for many rows: persistent CTAs that stream their rows through shared memory.
//
// The operator moves x and the residual in and h and y out, 8 bytes an element in 16-bit types, and is bound by HBM as long as
// an SM always has some 50 KB of loads under way and spends less than about 20 instructions an element.  Hence: a CTA owns a
// contiguous block of rows and keeps the next ones in flight with bulk copies (one thread, two instructions a row, no
// registers), while the current row goes from shared memory to registers, through its one or two norms and out; types are
// compile-time, and the arithmetic is two values an instruction.  The kernel that loads a row per CTA straight into registers
// (block_ops.cuh) measured 310 us on 16384 x 8192 with both norms and a gate: 43 instructions an element, and nothing in flight
// while a row is reduced.
//
// Rows that start on any address are copied from the 16-byte boundary below to the one above, and read element by element.
#pragma once
#include "block_ops.cuh"

namespace b200 {

struct NormStreamLayout
{
    unsigned x_bytes, r_bytes; // shared memory of one row, multiples of 16
    unsigned stages;
    WaitReport report;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t w)
{
    if(DT == OUT_BF16)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// eight (VEC = 8) or one (VEC = 1) consecutive elements of compile-time type as pairs
template <int DT, int VEC>
__device__ __forceinline__ void rd_vec(const uint8_t* p, float2 (&v)[VEC == 8 ? 4 : 1])
{
    if constexpr(VEC == 1)
        v[0] = make_float2(DT == OUT_F32 ? *reinterpret_cast<const float*>(p) : dec16(*reinterpret_cast<const uint16_t*>(p), DT), 0.f);
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
__device__ __forceinline__ void wr_vec(uint8_t* p, const float2 (&v)[VEC == 8 ? 4 : 1])
{
    if constexpr(VEC == 1)
    {
        if constexpr(DT == OUT_F32)
            *reinterpret_cast<float*>(p) = v[0].x;
        else
            *reinterpret_cast<uint16_t*>(p) = cvt_out16(v[0].x, DT == OUT_F16);
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
__host__ __device__ constexpr int esize_of(int dt) { return dt == OUT_F32 ? 4 : 2; }

// XD, RD: types of x and of the residual and h; PD: of every parameter of more than one value.  A thread holds CNT vectors of VEC
// elements, vector j at element (j * threads + t) * VEC.
template <int XD, int RD, int PD, int VEC, int CNT>
__global__ void __launch_bounds__(512, VEC * CNT <= 16 ? 2 : 1) norm_stream_kernel(const __grid_constant__ NormParams prm, const __grid_constant__ NormStreamLayout lay)
{
    constexpr int P = VEC == 8 ? 4 : 1; // pairs of a vector (VEC = 1: one value in the first half)
    constexpr int XS = esize_of(XD), RS = esize_of(RD), PS = esize_of(PD);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float red[8][32]; // two sets of slots, for even and odd rows: one barrier a sum is enough
    __shared__ __align__(8) uint64_t full[4];
    const unsigned t = threadIdx.x, T = blockDim.x, n = prm.n;
    const bool has_res = prm.res.ptr != nullptr;
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
    const uint8_t* const xg = static_cast<const uint8_t*>(prm.x.ptr);
    const uint8_t* const rg = static_cast<const uint8_t*>(prm.res.ptr);
    auto load = [&](unsigned i) { // row row0 + i into stage i % S, by one thread
        const unsigned s   = i % S;
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem) + s * stage_bytes;
        const uint8_t* xp  = xg + static_cast<size_t>(row0 + i) * prm.x.ld * XS;
        const unsigned xo  = VEC == 8 ? 0u : static_cast<unsigned>(reinterpret_cast<uintptr_t>(xp) & 15);
        const unsigned xb  = (xo + n * XS + 15u) & ~15u;
        unsigned rb        = 0;
        const uint8_t* rp  = nullptr;
        if(has_res)
        {
            rp = rg + static_cast<size_t>(row0 + i) * prm.res.ld * RS;
            const unsigned ro = VEC == 8 ? 0u : static_cast<unsigned>(reinterpret_cast<uintptr_t>(rp) & 15);
            rb                = (ro + n * RS + 15u) & ~15u;
            rp -= ro;
        }
        mbar_arrive_expect_tx(bar, xb + rb);
        bulk_load(dst, xp - xo, xb, bar);
        if(has_res)
            bulk_load(dst + lay.x_bytes, rp, rb, bar);
    };
    if(t == 0)
        for(unsigned i = 0; i < min(S, rows); ++i)
            load(i);
    unsigned s = 0, phase = 0;
    bool expired = false;
    for(unsigned i = 0; i < rows; ++i)
    {
        const unsigned row = row0 + i;
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
        if(VEC == 1)
        {
            xs += (reinterpret_cast<uintptr_t>(xg) + static_cast<size_t>(row) * prm.x.ld * XS) & 15;
            rs += (reinterpret_cast<uintptr_t>(rg) + static_cast<size_t>(row) * prm.res.ld * RS) & 15;
        }
        float2 h[CNT][P];
#pragma unroll
        for(int j = 0; j < CNT; ++j)
        {
            const unsigned col = (j * T + t) * VEC;
            if(col < n)
                rd_vec<XD, VEC>(xs + col * XS, h[j]);
            else
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = make_float2(0.f, 0.f);
        }
        auto stats = [&](int slot, float& mean, float& rstd) {
            slot += 4 * static_cast<int>(i & 1);
            mean = 0.f;
            if(prm.layer)
            {
                float2 a = make_float2(0.f, 0.f);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        a = __fadd2_rn(a, h[j][k]);
                mean = row_sum(a.x + a.y, red, slot) * prm.inv_n;
            }
            float2 a       = make_float2(0.f, 0.f);
            const float2 m = make_float2(-mean, VEC == 1 ? 0.f : -mean);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
                if((j * T + t) * VEC < n)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                    {
                        const float2 d = __fadd2_rn(h[j][k], m);
                        a              = __ffma2_rn(d, d, a);
                    }
            rstd = rsqrtf(row_sum(a.x + a.y, red, slot + 1) * prm.inv_n + prm.eps);
        };
        float mean = 0.f, rstd = 1.f;
        if(prm.post)
            stats(0, mean, rstd);
        const uint8_t* const pw = static_cast<const uint8_t*>(prm.post_weight.ptr) + param_at(prm.post_weight, row) * PS;
        const uint8_t* const pb = static_cast<const uint8_t*>(prm.post_bias.ptr) + param_at(prm.post_bias, row) * PS;
        const uint8_t* const pg = static_cast<const uint8_t*>(prm.gate.ptr) + param_at(prm.gate, row) * PS;
        const float gate1 = (prm.gate.ptr != nullptr && prm.gate_scalar) ? load_elem_any(prm.gate.ptr, prm.gate.dt, param_at(prm.gate, row)) : 1.f;
#pragma unroll
        for(int j = 0; j < CNT; ++j)
        {
            const unsigned col = (j * T + t) * VEC;
            if(col < n)
            {
                float2 q[P];
                if(prm.post)
                {
                    const float2 a = make_float2(rstd, rstd), b = make_float2(-mean, -mean);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __fmul2_rn(__fadd2_rn(h[j][k], b), a);
                    if(prm.post_weight.ptr != nullptr)
                    {
                        rd_vec<PD, VEC>(pw + col * PS, q);
#pragma unroll
                        for(int k = 0; k < P; ++k)
                            h[j][k] = __fmul2_rn(h[j][k], q[k]);
                    }
                    if(prm.post_bias.ptr != nullptr)
                    {
                        rd_vec<PD, VEC>(pb + col * PS, q);
#pragma unroll
                        for(int k = 0; k < P; ++k)
                            h[j][k] = __fadd2_rn(h[j][k], q[k]);
                    }
                }
                if(prm.gate.ptr != nullptr)
                {
                    if(prm.gate_scalar)
#pragma unroll
                        for(int k = 0; k < P; ++k)
                            q[k] = make_float2(gate1, gate1);
                    else
                        rd_vec<PD, VEC>(pg + col * PS, q);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __fmul2_rn(h[j][k], q[k]);
                }
                if(has_res)
                {
                    const float2 a = make_float2(prm.res_scale, prm.res_scale);
                    rd_vec<RD, VEC>(rs + col * RS, q);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __ffma2_rn(a, q[k], h[j][k]);
                }
                if(prm.h.ptr != nullptr)
                    wr_vec<RD, VEC>(static_cast<uint8_t*>(prm.h.ptr) + (static_cast<size_t>(row) * prm.h.ld + col) * RS, h[j]);
                if(VEC == 1)
                    h[j][0].y = 0.f;
            }
        }
        stats(2, mean, rstd);
        // every thread has read its part of the stage (the sum's barrier): the row after next may land there
        if(T == 32)
            __syncwarp();
        if(t == 0 && i + S < rows && !expired)
            load(i + S);
        if(++s == S)
        {
            s = 0;
            phase ^= 1u;
        }
        const uint8_t* const w = static_cast<const uint8_t*>(prm.weight.ptr) + param_at(prm.weight, row) * PS;
        const uint8_t* const b = static_cast<const uint8_t*>(prm.bias.ptr) + param_at(prm.bias, row) * PS;
#pragma unroll
        for(int j = 0; j < CNT; ++j)
        {
            const unsigned col = (j * T + t) * VEC;
            if(col < n)
            {
                const float2 a = make_float2(rstd, rstd), m = make_float2(-mean, -mean), o = make_float2(prm.weight_offset, prm.weight_offset);
                float2 q[P];
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = __fmul2_rn(__fadd2_rn(h[j][k], m), a);
                if(prm.weight.ptr != nullptr)
                {
                    rd_vec<PD, VEC>(w + col * PS, q);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __fmul2_rn(h[j][k], __fadd2_rn(q[k], o));
                }
                if(prm.bias.ptr != nullptr)
                {
                    rd_vec<PD, VEC>(b + col * PS, q);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = __fadd2_rn(h[j][k], q[k]);
                }
            }
        }
        // one test of y's type a row
        uint8_t* const y = static_cast<uint8_t*>(prm.y.ptr) + static_cast<size_t>(row) * prm.y.ld * bytes_of_mode(prm.y.dt);
        auto store_all   = [&](auto tag) {
            constexpr int YD = decltype(tag)::value;
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = (j * T + t) * VEC;
                if(col < n)
                    wr_vec<YD, VEC>(y + col * esize_of(YD), h[j]);
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
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = (j * T + t) * VEC;
                const float f[8]   = {h[j][0].x, h[j][0].y, h[j][1].x, h[j][1].y, h[j][2].x, h[j][2].y, h[j][3].x, h[j][3].y};
                emit<8>(prm, row, col, col < n, f);
            }
            fill_scale_padding(prm.sf, row, prm.M, n >> 5, t, T);
        }
    }
    if(expired)
    {
        // copies still in flight land before this CTA's shared memory is released (bounded)
        const uint64_t t0 = global_timer_ns();
        while(global_timer_ns() - t0 < 200000ull) {}
    }
}

} // namespace b200
