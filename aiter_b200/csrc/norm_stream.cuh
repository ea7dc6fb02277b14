// gated_residual_norm for many rows: persistent CTAs that stream their rows through shared memory.
//
// The operator moves x and the residual in and h and y out, 8 bytes an element in 16-bit types, and is bound by HBM as long as
// an SM always has some 50 KB of loads under way and spends few instructions an element (35 with both norms and a gate: 16384 x 8192
// 184 us, 5.8 TB/s).  Hence: a CTA owns a contiguous block of rows and keeps the next ones in flight with bulk copies (one thread,
// two instructions a row, no registers), while the current row goes from shared memory to registers, through its one or two norms
// and out; a thread holds 16 values, over which the fixed work of a row (its sums, addresses) is spread, and types are compile-time.
//
// Rows of any width have a kernel of their own below, short rows another.
#pragma once
#include "block_ops.cuh"

namespace b200 {

// (Two scalar instructions each: the two-wide forms measured slower here, 16384 x 8192 with both norms and a gate 196 against
// 178 us - the values come in and go out one by one, and the pairs cost moves.)
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }

struct NormStreamLayout
{
    unsigned x_bytes, r_bytes; // shared memory of one row, multiples of 16
    unsigned stages;
    unsigned param_off;        // rows of any width: where the current parameters are kept, param_pitch bytes each
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
// eight consecutive elements of a compile-time type, aligned to the vector, as pairs
template <int DT>
__device__ __forceinline__ void rd_vec(const uint8_t* p, float2 (&v)[4])
{
    if constexpr(DT == OUT_F32)
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
template <int DT>
__device__ __forceinline__ void wr_vec(uint8_t* p, const float2 (&v)[4])
{
    if constexpr(DT == OUT_F32)
    {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    }
    else
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_out16x2(v[0].x, v[0].y, DT == OUT_F16), pack_out16x2(v[1].x, v[1].y, DT == OUT_F16),
                                                  pack_out16x2(v[2].x, v[2].y, DT == OUT_F16), pack_out16x2(v[3].x, v[3].y, DT == OUT_F16));
}

// h *= offset + p  and  h += p for a parameter vector p of the row
template <int PD, int CNT, bool FULL = false>
__device__ __forceinline__ void scale_by(float2 (&h)[CNT][4], const uint8_t* p, unsigned col0, unsigned col_step, unsigned n, float offset)
{
    const float2 o = make_float2(offset, offset);
    const bool plain = offset == 0.f;
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        const unsigned col = col0 + j * col_step;
        if(FULL || col < n)
        {
            float2 q[4];
            rd_vec<PD>(p + col * esize_of(PD), q);
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[j][k] = mul2(h[j][k], plain ? q[k] : add2(q[k], o));
        }
    }
}
template <int PD, int CNT, bool FULL = false>
__device__ __forceinline__ void shift_by(float2 (&h)[CNT][4], const uint8_t* p, unsigned col0, unsigned col_step, unsigned n)
{
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        const unsigned col = col0 + j * col_step;
        if(FULL || col < n)
        {
            float2 q[4];
            rd_vec<PD>(p + col * esize_of(PD), q);
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[j][k] = add2(h[j][k], q[k]);
        }
    }
}
// the row's vectors as an MX operand
template <bool FP4, int CNT, bool FULL = false>
__device__ __forceinline__ void emit_mx(const BlockScales& sf, uint8_t* y, unsigned row, unsigned col0, unsigned col_step, unsigned n, const float2 (&h)[CNT][4])
{
    uint8_t* const sf_row = sf.ptr + sf_offset(sf, row, 0); // (block 0; the others lie at offsets that do not depend on the row)
#pragma unroll
    for(int j = 0; j < CNT; ++j)
    {
        const unsigned col = col0 + j * col_step;
        const bool in      = FULL || col < n;
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

// XD, RD: types of x and of the residual and h; PD: of every parameter of more than one value.  A thread holds CNT vectors of eight
// elements, vector j at element (j * threads + t) * 8; FULL: exactly the row, no vector lies behind it.
template <int XD, int RD, int PD, int CNT, bool FULL>
__global__ void __launch_bounds__(512, CNT <= 2 ? 2 : 1) norm_stream_kernel(const __grid_constant__ NormParams prm, const __grid_constant__ NormStreamLayout lay)
{
    constexpr int P = 4;
    constexpr int XS = esize_of(XD), RS = esize_of(RD), PS = esize_of(PD);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float red[8][32]; // two sets of slots, for even and odd rows: one barrier a sum is enough
    __shared__ __align__(8) uint64_t full[4];
    __shared__ volatile unsigned gave_up; // 1 + the row in which a thread's wait ran out
    const unsigned t = threadIdx.x, T = blockDim.x, n = prm.n;
    const bool has_res = prm.res.ptr != nullptr;
    const bool gate_one = prm.gate.ptr != nullptr && prm.gate_scalar;
    // this CTA's rows: the first `extra` CTAs take one more
    const unsigned per = prm.M / gridDim.x, extra = prm.M % gridDim.x;
    const unsigned row0 = blockIdx.x * per + min(blockIdx.x, extra);
    const unsigned rows = per + (blockIdx.x < extra ? 1u : 0u);
    const unsigned S = lay.stages, stage_bytes = lay.x_bytes + lay.r_bytes;
    if(t == 0)
    {
        gave_up = 0;
        for(unsigned s = 0; s < S; ++s)
            mbar_init(smem_u32(&full[s]), 1);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    auto load = [&](unsigned row, unsigned s) { // a row into stage s, by one thread
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem) + s * stage_bytes;
        mbar_arrive_expect_tx(bar, stage_bytes);
        bulk_load(dst, static_cast<const uint8_t*>(prm.x.ptr) + static_cast<size_t>(row) * prm.x.ld * XS, lay.x_bytes, bar);
        if(has_res)
            bulk_load(dst + lay.x_bytes, static_cast<const uint8_t*>(prm.res.ptr) + static_cast<size_t>(row) * prm.res.ld * RS, lay.r_bytes, bar);
    };
    if(t == 0 && lay.report.withhold == 0u)
        for(unsigned i = 0; i < min(S, rows); ++i)
            load(row0 + i, i);
    // the parameters' entries of the current row, until row `change`: indexes, since registers are what two CTAs an SM leave
    // short (addresses are formed where they are used, from the parameter bank)
    unsigned ew = 0, eb = 0, epw = 0, epb = 0, eg = 0, change = 0;
    float gate1  = 1.f;
    auto entries = [&](unsigned row) {
        change    = 0xFFFFFFFFu;
        auto take = [&](const RowParam& q) {
            if(q.ld == 0)
                return 0u;
            const unsigned e = row / q.rows_per;
            change           = min(change, (e + 1) * q.rows_per);
            return e;
        };
        ew  = take(prm.weight);
        eb  = take(prm.bias);
        epw = take(prm.post_weight);
        epb = take(prm.post_bias);
        eg  = take(prm.gate);
        if(gate_one)
            gate1 = load_elem_any(prm.gate.ptr, prm.gate.dt, static_cast<size_t>(eg) * prm.gate.ld);
    };
    auto entry = [&](const RowParam& q, unsigned e) { return static_cast<const uint8_t*>(q.ptr) + static_cast<size_t>(e) * q.ld * PS; };
    unsigned s = 0, phase = 0;
    bool stopped = false;
    const unsigned col0 = t * 8, col_step = T * 8;
#pragma unroll 1
    for(unsigned i = 0; i < rows; ++i)
    {
        const unsigned row = row0 + i;
        if(row >= change) // (the same for every thread)
            entries(row);
        // Bounded, though a copy of valid memory always completes.  A thread whose wait runs out stores no h and adds a NaN to the row's
        // sum; a row with a NaN asks, behind the sum's barrier, whether that was the reason, and then the whole CTA stops there.  The
        // status record says that the output is incomplete.
        bool late = false; // this thread's wait ran out
        if(!mbar_try_wait(smem_u32(&full[s]), phase))
        {
            const uint64_t t0 = global_timer_ns();
            while(!late && !mbar_try_wait_parked(smem_u32(&full[s]), phase, kParkNs))
                late = global_timer_ns() - t0 > lay.report.limit_ns;
            if(late)
            {
                gave_up = i + 1;
                report_timeout(lay.report, ST_TIMEOUT_ROWS, i);
            }
        }
        const uint8_t* xs = smem + s * stage_bytes;
        const uint8_t* rs = xs + lay.x_bytes;
        float2 h[CNT][P];
        {
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(FULL || col < n)
                    rd_vec<XD>(xs + col * XS, h[j]);
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
                        a = add2(a, h[j][k]);
                mean = row_sum(a.x + a.y, red, slot) * prm.inv_n;
                a    = make_float2(0.f, 0.f);
                const float2 m = make_float2(-mean, -mean);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
                {
                    const unsigned col = col0 + j * col_step;
                    if(FULL || col < n)
#pragma unroll
                        for(int k = 0; k < P; ++k)
                        {
                            const float2 d = add2(h[j][k], m);
                            a = fma2(d, d, a);
                        }
                }
            }
            else
            {
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        a = fma2(h[j][k], h[j][k], a);
            }
            rstd = rsqrtf(row_sum(late ? __uint_as_float(0x7FFFFFFFu) : a.x + a.y, red, slot + 1) * prm.inv_n + prm.eps);
        };
        float mean = 0.f, rstd = 1.f;
        if(prm.post)
        {
            stats(0, mean, rstd);
            if(rstd != rstd && gave_up == i + 1)
            {
                stopped = true;
                break;
            }
            const float2 a = make_float2(rstd, rstd);
            if(prm.layer)
            {
                const float2 m = make_float2(-mean, -mean);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = add2(h[j][k], m);
            }
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = mul2(h[j][k], a);
            if(prm.post_weight.ptr != nullptr)
                scale_by<PD, CNT, FULL>(h, entry(prm.post_weight, epw), col0, col_step, n, 0.f);
            if(prm.post_bias.ptr != nullptr)
                shift_by<PD, CNT, FULL>(h, entry(prm.post_bias, epb), col0, col_step, n);
        }
        if(prm.gate.ptr != nullptr && !prm.gate_scalar)
            scale_by<PD, CNT, FULL>(h, entry(prm.gate, eg), col0, col_step, n, 0.f);
        else if(gate_one)
        {
            const float2 a = make_float2(gate1, gate1);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = mul2(h[j][k], a);
        }
        if(has_res)
        {
            const float2 a = make_float2(prm.res_scale, prm.res_scale);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(FULL || col < n)
                {
                    float2 q[P];
                    rd_vec<RD>(rs + col * RS, q);
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = fma2(a, q[k], h[j][k]);
                }
            }
        }
        // elements behind the row count for nothing in the sums (a first layer norm or its bias has touched them)
        if(!FULL && prm.post)
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(col >= n)
#pragma unroll
                    for(int k = 0; k < P; ++k)
                        h[j][k] = make_float2(0.f, 0.f);
            }
        if(prm.h.ptr != nullptr && !late)
        {
            uint8_t* const hg = static_cast<uint8_t*>(prm.h.ptr) + static_cast<size_t>(row) * prm.h.ld * RS;
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(FULL || col < n)
                    wr_vec<RD>(hg + col * RS, h[j]);
            }
        }
        stats(2, mean, rstd);
        if(rstd != rstd && gave_up == i + 1)
        {
            stopped = true;
            break;
        }
        // every thread has read its part of the stage (the sum's barrier): a later row may land there
        if(t == 0 && i + S < rows)
            load(row + S, s);
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
                        h[j][k] = add2(h[j][k], m);
            }
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < P; ++k)
                    h[j][k] = mul2(h[j][k], a);
        }
        if(prm.weight.ptr != nullptr)
            scale_by<PD, CNT, FULL>(h, entry(prm.weight, ew), col0, col_step, n, prm.weight_offset);
        if(prm.bias.ptr != nullptr)
            shift_by<PD, CNT, FULL>(h, entry(prm.bias, eb), col0, col_step, n);
        // one test of y's type a row
        uint8_t* const yg = static_cast<uint8_t*>(prm.y.ptr) + static_cast<size_t>(row) * prm.y.ld * bytes_of_mode(prm.y.dt);
        auto store_all = [&](auto tag) {
            constexpr int YD = decltype(tag)::value;
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned col = col0 + j * col_step;
                if(FULL || col < n)
                    wr_vec<YD>(yg + col * esize_of(YD), h[j]);
            }
        };
        if(prm.y.dt == OUT_BF16)
            store_all(std::integral_constant<int, OUT_BF16>{});
        else if(prm.y.dt == OUT_F16)
            store_all(std::integral_constant<int, OUT_F16>{});
        else if(prm.y.dt == OUT_F32)
            store_all(std::integral_constant<int, OUT_F32>{});
        else
        {
            if(prm.y.dt == OUT_E2M1)
                emit_mx<true, CNT, FULL>(prm.sf, yg, row, col0, col_step, n, h);
            else
                emit_mx<false, CNT, FULL>(prm.sf, yg, row, col0, col_step, n, h);
            if(prm.sf.layout != QSL_PLAIN && (row == prm.M - 1 || (n & 255) != 0))
                fill_scale_padding(prm.sf, row, prm.M, n >> 5, t, T);
        }
    }
    if(stopped)
    {
        // copies still in flight land before this CTA's shared memory is released (bounded)
        const uint64_t t0 = global_timer_ns();
        while(global_timer_ns() - t0 < 200000ull) {}
    }
}

// Rows of any width of dense tensors: row r starts at element r * ld, and with equal pitches (modulo 8) and aligned bases the
// groups of eight elements that are aligned in one tensor are aligned in all.  A thread takes such groups - the first and the last
// of a row only in part -, so every access of x, residual, h and y stays a 16-byte one.  A row's phase in its groups repeats every
// eight rows: a CTA takes every eighth row of its block, and keeps the parameters in shared memory at that phase.  (One element a
// lane at a time: 8192 x 4097 106 to 150 us, at about 100 instructions an element; parameters shifted into place by selects on
// every row, 8200 x 1155 with three of them, 55 us.  As it stands: 8192 x 4097 54 us, 8200 x 1155 with three 40, at 77 instructions an
// element - a thread holds eight values there, over which the row's two sums and its addresses are spread.)
template <int XD, int RD, int PD, int CNT>
__global__ void __launch_bounds__(512, 2) norm_stream_flat_kernel(const __grid_constant__ NormParams prm, const __grid_constant__ NormStreamLayout lay)
{
    constexpr int XS = esize_of(XD), RS = esize_of(RD), PS = esize_of(PD);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float red[8][32];
    __shared__ __align__(8) uint64_t full[4];
    __shared__ volatile unsigned gave_up; // 1 + the row in which a thread's wait ran out
    const unsigned t = threadIdx.x, T = blockDim.x, n = prm.n;
    const bool has_res  = prm.res.ptr != nullptr;
    const bool gate_one = prm.gate.ptr != nullptr && prm.gate_scalar;
    // this CTA's rows: row_of(0), row_of(1), ... of one residue class modulo 8 (the grid is a multiple of 8)
    const unsigned cls = blockIdx.x & 7, of_class = prm.M > cls ? (prm.M - cls + 7) / 8 : 0;
    const unsigned team = gridDim.x / 8, mate = blockIdx.x / 8;
    const unsigned per = of_class / team, extra = of_class % team;
    const unsigned row0 = cls + 8 * (mate * per + min(mate, extra));
    const unsigned rows = per + (mate < extra ? 1u : 0u);
    auto row_of         = [&](unsigned i) { return row0 + 8 * i; };
    const unsigned S = lay.stages, stage_bytes = lay.x_bytes + lay.r_bytes;
    if(t == 0)
    {
        gave_up = 0;
        for(unsigned s = 0; s < S; ++s)
            mbar_init(smem_u32(&full[s]), 1);
        mbar_fence_init();
        fence_proxy_async_smem();
    }
    __syncthreads();
    grid_dependency_wait();
    grid_launch_dependents();
    // first element of this CTA's rows within their groups of eight (the same in every tensor): the row is elements [e8, end)
    const unsigned e8 = static_cast<unsigned>((reinterpret_cast<uintptr_t>(prm.x.ptr) / XS + static_cast<size_t>(row0) * prm.x.ld) & 7), end = e8 + n;
    auto load     = [&](unsigned row, unsigned s) { // whole groups of a row into stage s, by one thread
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem) + s * stage_bytes;
        // the 16-byte pieces that hold something of the row, at their places in its groups
        const unsigned x0 = (e8 * XS) & ~15u, xb = (((e8 + n) * XS + 15) & ~15u) - x0;
        const unsigned r0 = (e8 * RS) & ~15u, rb = (((e8 + n) * RS + 15) & ~15u) - r0;
        mbar_arrive_expect_tx(bar, xb + (has_res ? rb : 0u));
        bulk_load(dst + x0, static_cast<const uint8_t*>(prm.x.ptr) + (static_cast<size_t>(row) * prm.x.ld - e8) * XS + x0, xb, bar);
        if(has_res)
            bulk_load(dst + lay.x_bytes + r0, static_cast<const uint8_t*>(prm.res.ptr) + (static_cast<size_t>(row) * prm.res.ld - e8) * RS + r0, rb, bar);
    };
    if(t == 0 && lay.report.withhold == 0u)
        for(unsigned i = 0; i < min(S, rows); ++i)
            load(row_of(i), i);
    // the parameters of the current entries, element e of each at place e8 + e, until row `change`
    uint8_t* const params = smem + lay.param_off;
    float gate1           = 1.f;
    unsigned change       = 0;
    auto entries          = [&](unsigned row) {
        change    = 0xFFFFFFFFu;
        int k     = 0;
        auto take = [&](const RowParam& q) {
            if(q.ptr == nullptr)
                return;
            if(q.ld != 0)
                change = min(change, (row / q.rows_per + 1) * q.rows_per);
            using E      = std::conditional_t<PD == OUT_F32, uint32_t, uint16_t>;
            const E* src = static_cast<const E*>(q.ptr) + param_at(q, row);
            E* dst       = reinterpret_cast<E*>(params + (k++) * lay.param_pitch) + e8;
            for(unsigned e = t; e < n; e += T)
                dst[e] = src[e];
        };
        __syncthreads(); // nobody reads the previous entries any more
        take(prm.weight);
        take(prm.bias);
        take(prm.post_weight);
        take(prm.post_bias);
        if(!gate_one)
            take(prm.gate);
        else
        {
            if(prm.gate.ld != 0)
                change = min(change, (row / prm.gate.rows_per + 1) * prm.gate.rows_per);
            gate1 = load_elem_any(prm.gate.ptr, prm.gate.dt, param_at(prm.gate, row));
        }
        __syncthreads();
    };
    // where each parameter lies (the order of `take`)
    int slots      = 0;
    auto slot      = [&](const RowParam& q) { return q.ptr != nullptr ? slots++ : -1; };
    const int at_w = slot(prm.weight), at_b = slot(prm.bias), at_pw = slot(prm.post_weight), at_pb = slot(prm.post_bias);
    const int at_g = gate_one ? -1 : slot(prm.gate);
    const unsigned col0 = t * 8, col_step = T * 8;
    auto place = [&](int at) { return params + at * lay.param_pitch; };
    unsigned s = 0, phase = 0;
    bool stopped = false;
#pragma unroll 1
    for(unsigned i = 0; i < rows; ++i)
    {
        const unsigned row = row_of(i);
        if(row >= change) // (the same for every thread)
            entries(row);
        bool late = false; // this thread's wait ran out
        if(!mbar_try_wait(smem_u32(&full[s]), phase))
        {
            const uint64_t t0 = global_timer_ns();
            while(!late && !mbar_try_wait_parked(smem_u32(&full[s]), phase, kParkNs))
                late = global_timer_ns() - t0 > lay.report.limit_ns;
            if(late)
            {
                gave_up = i + 1;
                report_timeout(lay.report, ST_TIMEOUT_ROWS, i);
            }
        }
        const uint8_t* xs = smem + s * stage_bytes;
        const uint8_t* rs = xs + lay.x_bytes;
        auto group   = [&](int j) { return j * T + t; };
        auto whole   = [&](unsigned v) { return (v != 0 || e8 == 0) && 8 * v + 8 <= end; };
        auto exists  = [&](unsigned v) { return 8 * v < end; };
        auto for_row = [&](unsigned v, auto&& f) { // the elements of a group that is only partly the row's
#pragma unroll
            for(int k = 0; k < 8; ++k)
                if(8 * v + k >= e8 && 8 * v + k < end)
                    f(k);
        };
        float2 h[CNT][4];
        auto clear_outside = [&](unsigned v, float2 (&g)[4]) {
#pragma unroll
            for(int k = 0; k < 4; ++k)
                g[k] = make_float2((8 * v + 2 * k >= e8 && 8 * v + 2 * k < end) ? g[k].x : 0.f, (8 * v + 2 * k + 1 >= e8 && 8 * v + 2 * k + 1 < end) ? g[k].y : 0.f);
        };
#pragma unroll
        for(int j = 0; j < CNT; ++j)
        {
            const unsigned v = group(j);
            if(exists(v))
            {
                rd_vec<XD>(xs + v * (8 * XS), h[j]);
                if(!whole(v))
                    clear_outside(v, h[j]);
            }
            else
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    h[j][k] = make_float2(0.f, 0.f);
        }
        auto stats = [&](int slot_, float& mean, float& rstd) {
            slot_ += 4 * static_cast<int>(i & 1);
            float2 a = make_float2(0.f, 0.f);
            mean     = 0.f;
            if(prm.layer)
            {
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                        a = add2(a, h[j][k]);
                mean = row_sum(a.x + a.y, red, slot_) * prm.inv_n;
                a    = make_float2(0.f, 0.f);
                const float2 m = make_float2(-mean, -mean);
#pragma unroll
                for(int j = 0; j < CNT; ++j)
                {
                    const unsigned v = group(j);
                    float2 d[4];
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                        d[k] = add2(h[j][k], m);
                    if(!whole(v))
                        clear_outside(v, d);
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                        a = fma2(d[k], d[k], a);
                }
            }
            else
            {
#pragma unroll
                for(int j = 0; j < CNT; ++j)
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                        a = fma2(h[j][k], h[j][k], a);
            }
            rstd = rsqrtf(row_sum(late ? __uint_as_float(0x7FFFFFFFu) : a.x + a.y, red, slot_ + 1) * prm.inv_n + prm.eps);
        };
        auto scale1 = [&](float f) {
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    h[j][k] = mul2(h[j][k], make_float2(f, f));
        };
        auto shift1 = [&](float f) {
#pragma unroll
            for(int j = 0; j < CNT; ++j)
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    h[j][k] = add2(h[j][k], make_float2(f, f));
        };
        float mean = 0.f, rstd = 1.f;
        if(prm.post)
        {
            stats(0, mean, rstd);
            if(rstd != rstd && gave_up == i + 1)
            {
                stopped = true;
                break;
            }
            if(prm.layer)
                shift1(-mean);
            scale1(rstd);
            if(at_pw >= 0)
                scale_by<PD, CNT>(h, place(at_pw), col0, col_step, end, 0.f);
            if(at_pb >= 0)
                shift_by<PD, CNT>(h, place(at_pb), col0, col_step, end);
        }
        if(at_g >= 0)
            scale_by<PD, CNT>(h, place(at_g), col0, col_step, end, 0.f);
        else if(gate_one)
            scale1(gate1);
        if(has_res)
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned v = group(j);
                if(exists(v))
                {
                    float2 q[4];
                    rd_vec<RD>(rs + v * (8 * RS), q);
#pragma unroll
                    for(int k = 0; k < 4; ++k)
                        h[j][k] = fma2(make_float2(prm.res_scale, prm.res_scale), q[k], h[j][k]);
                }
            }
        // values outside the row count for nothing in the sums
#pragma unroll
        for(int j = 0; j < CNT; ++j)
            if(!whole(group(j)))
                clear_outside(group(j), h[j]);
        auto store = [&](const RowTensor& y, auto tag) {
            constexpr int DT = decltype(tag)::value;
            uint8_t* const p = static_cast<uint8_t*>(y.ptr) + (static_cast<size_t>(row) * y.ld - e8) * esize_of(DT);
#pragma unroll
            for(int j = 0; j < CNT; ++j)
            {
                const unsigned v = group(j);
                if(whole(v))
                    wr_vec<DT>(p + v * (8 * esize_of(DT)), h[j]);
                else if(exists(v))
                    for_row(v, [&](int k) { store_out(p, 8 * v + k, (k & 1) ? h[j][k / 2].y : h[j][k / 2].x, DT); });
            }
        };
        if(prm.h.ptr != nullptr && !late)
            store(prm.h, std::integral_constant<int, RD>{});
        stats(2, mean, rstd);
        if(rstd != rstd && gave_up == i + 1)
        {
            stopped = true;
            break;
        }
        // every thread has read its part of the stage (the sum's barrier): a later row may land there
        if(t == 0 && i + S < rows)
            load(row_of(i + S), s);
        if(++s == S)
        {
            s = 0;
            phase ^= 1u;
        }
        if(prm.layer)
            shift1(-mean);
        scale1(rstd);
        if(at_w >= 0)
            scale_by<PD, CNT>(h, place(at_w), col0, col_step, end, prm.weight_offset);
        if(at_b >= 0)
            shift_by<PD, CNT>(h, place(at_b), col0, col_step, end);
        if(prm.y.dt == OUT_BF16)
            store(prm.y, std::integral_constant<int, OUT_BF16>{});
        else if(prm.y.dt == OUT_F16)
            store(prm.y, std::integral_constant<int, OUT_F16>{});
        else
            store(prm.y, std::integral_constant<int, OUT_F32>{});
    }
    if(stopped)
    {
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
                    const float2 d = add2(h[0][k], m);
                    a              = fma2(d, d, a);
                }
            rstd = rsqrtf(sum(a.x + a.y) * prm.inv_n + prm.eps);
        };
        auto normalise = [&](float mean, float rstd) {
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[0][k] = mul2(add2(h[0][k], make_float2(-mean, -mean)), make_float2(rstd, rstd));
        };
        auto entry = [&](const RowParam& q) { return static_cast<const uint8_t*>(q.ptr) + param_at(q, row) * PS; };
        float mean, rstd;
        if(prm.post)
        {
            stats(mean, rstd);
            normalise(mean, rstd);
            if(prm.post_weight.ptr != nullptr)
                scale_by<PD, 1>(h, entry(prm.post_weight), col, 0, n, 0.f);
            if(prm.post_bias.ptr != nullptr)
                shift_by<PD, 1>(h, entry(prm.post_bias), col, 0, n);
        }
        if(prm.gate.ptr != nullptr)
        {
            if(prm.gate_scalar)
            {
                const float g = load_elem_any(prm.gate.ptr, prm.gate.dt, param_at(prm.gate, row));
#pragma unroll
                for(int k = 0; k < 4; ++k)
                    h[0][k] = mul2(h[0][k], make_float2(g, g));
            }
            else
                scale_by<PD, 1>(h, entry(prm.gate), col, 0, n, 0.f);
        }
        if(has_res && in)
        {
            unpack<8, RD == OUT_F32>(cr, RD, v);
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[0][k] = fma2(make_float2(prm.res_scale, prm.res_scale), make_float2(v[2 * k], v[2 * k + 1]), h[0][k]);
        }
        if(!in)
#pragma unroll
            for(int k = 0; k < 4; ++k)
                h[0][k] = make_float2(0.f, 0.f);
        if(prm.h.ptr != nullptr && in)
            wr_vec<RD>(static_cast<uint8_t*>(prm.h.ptr) + (static_cast<size_t>(row) * prm.h.ld + col) * RS, h[0]);
        stats(mean, rstd);
        normalise(mean, rstd);
        if(prm.weight.ptr != nullptr)
            scale_by<PD, 1>(h, entry(prm.weight), col, 0, n, prm.weight_offset);
        if(prm.bias.ptr != nullptr)
            shift_by<PD, 1>(h, entry(prm.bias), col, 0, n);
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
                wr_vec<OUT_BF16>(y + col * 2, h[0]);
            else if(prm.y.dt == OUT_F16)
                wr_vec<OUT_F16>(y + col * 2, h[0]);
            else
                wr_vec<OUT_F32>(y + col * 4, h[0]);
        }
    }
}

} // namespace b200
