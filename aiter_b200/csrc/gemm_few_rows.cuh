// bf16 GEMM with a fused epilogue for one to four activation rows: act(A B^T + bias) + residual without tensor cores.
//
// The product is a stream of the weights through HBM, and what limits it is how early and how many of its loads are under way: a warp
// takes two columns (or a slice of their K, KS warps for it), eight 16-byte loads of weights a lane at a time, and a start-up of one
// block barrier or none - against the descriptors, barriers and TMEM of the tensor-core path (1 x 4096 x 4096 8.5 us against
// 10.0, 1 x 1024 x 8192 5.5 and 12.9, 1 x 464 x 512 2.4 and 4.2).  With more rows the fp32 multiply-adds show: the launch rule lets
// two to four rows come here for small weights only.
#pragma once
#include "activation.cuh"
#include "epilogue.cuh"
#include "gemm_common.cuh"

namespace b200 {

struct FewRowsParams
{
    const uint8_t* a; // [M, K] bf16
    const uint8_t* b; // [N, K] bf16
    long long a_ld, b_ld; // bytes between rows, multiples of 16
    const void* bias;
    const void* res;
    void* out;
    long long res_ld, out_ld;
    int bias_mode, res_mode, out_mode, act;
    unsigned N, K; // K a multiple of 8
};

constexpr int kFewRowsCols = 2; // columns of a warp: the activations are read and unpacked once for both

template <int M, int KS>
__global__ void __launch_bounds__(256) gemm_few_rows_kernel(const __grid_constant__ FewRowsParams prm)
{
    constexpr int C = kFewRowsCols, U = 4; // C x U loads of weights under way per lane
    __shared__ float red[8][M * C];
    const unsigned warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned col = (blockIdx.x * (8 / KS) + warp / KS) * C, slice = warp % KS;
    grid_dependency_wait();
    grid_launch_dependents();
    // lane m * C + c of the first slice finishes row m of column col + c
    const unsigned my_row = lane / C, my_col = col + lane % C;
    const bool finishes   = slice == 0 && lane < M * C && my_col < prm.N;
    float2 acc[M][C];
#pragma unroll
    for(int m = 0; m < M; ++m)
#pragma unroll
        for(int c = 0; c < C; ++c)
            acc[m][c] = make_float2(0.f, 0.f);
    float bias = 0.f, res = 0.f;
    const uint8_t* b = prm.b + static_cast<size_t>(col) * prm.b_ld;
    for(unsigned k0 = slice * 256 + lane * 8; k0 < prm.K; k0 += KS * 256 * U)
    {
        uint4 w[U][C];
#pragma unroll
        for(int u = 0; u < U; ++u)
        {
            const unsigned k = k0 + u * (KS * 256);
#pragma unroll
            for(int c = 0; c < C; ++c)
            {
                w[u][c] = make_uint4(0, 0, 0, 0);
                if(k < prm.K && col + c < prm.N)
                    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[u][c].x), "=r"(w[u][c].y), "=r"(w[u][c].z), "=r"(w[u][c].w) : "l"(b + c * prm.b_ld + k * 2ull));
            }
        }
#pragma unroll
        for(int u = 0; u < U; ++u)
        {
            const unsigned k = k0 + u * (KS * 256);
            if(k < prm.K)
            {
                float2 wf[C][4];
#pragma unroll
                for(int c = 0; c < C; ++c)
                {
                    const uint32_t ws[4] = {w[u][c].x, w[u][c].y, w[u][c].z, w[u][c].w};
#pragma unroll
                    for(int i = 0; i < 4; ++i)
                        wf[c][i] = make_float2(__uint_as_float(ws[i] << 16), __uint_as_float(ws[i] & 0xFFFF0000u));
                }
#pragma unroll
                for(int m = 0; m < M; ++m)
                {
                    const uint4 x        = *reinterpret_cast<const uint4*>(prm.a + m * prm.a_ld + k * 2ull);
                    const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for(int i = 0; i < 4; ++i)
                    {
                        const float2 xf = make_float2(__uint_as_float(xs[i] << 16), __uint_as_float(xs[i] & 0xFFFF0000u));
#pragma unroll
                        for(int c = 0; c < C; ++c)
                            acc[m][c] = __ffma2_rn(xf, wf[c][i], acc[m][c]);
                    }
                }
            }
        }
    }
    if(finishes)
    {
        if(prm.bias != nullptr)
            bias = load_elem(prm.bias, prm.bias_mode, my_col);
        if(prm.res != nullptr)
            res = load_elem(prm.res, prm.res_mode, static_cast<size_t>(my_row) * prm.res_ld + my_col);
    }
    float mine = 0.f;
#pragma unroll
    for(int m = 0; m < M; ++m)
#pragma unroll
        for(int c = 0; c < C; ++c)
        {
            float s = acc[m][c].x + acc[m][c].y;
#pragma unroll
            for(int d = 16; d > 0; d >>= 1)
                s += __shfl_xor_sync(0xffffffffu, s, d);
            if(static_cast<int>(lane) == m * C + c)
                mine = s;
        }
    if(KS > 1)
    {
        if(lane < M * C)
            red[warp][lane] = mine;
        __syncthreads();
        if(finishes)
        {
            mine = 0.f;
#pragma unroll
            for(int z = 0; z < KS; ++z)
                mine += red[warp + z][lane];
        }
    }
    if(finishes)
    {
        float v[1] = {mine + bias};
        activate(v, prm.act);
        store_out(prm.out, static_cast<size_t>(my_row) * prm.out_ld + my_col, v[0] + res, prm.out_mode);
    }
}

} // namespace b200
