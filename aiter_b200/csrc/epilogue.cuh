// Fused GEMM epilogue: out = act(A B^T + bias) + residual on the fp32 accumulator, rounded once.
//
// Row-major output tiles (activations on the 128-row slot) leave in steps of 32 columns, and EIGHT warps share them, two per
// TMEM lane quarter on alternating steps: an activation costs about 20 issue slots a value, a scheduler runs one warp of a
// quarter, and the accumulator of an MX tile 256 columns wide has no second one to hide behind.  Every epilogue warp owns two
// slots in shared memory: the residual's tile of a step is loaded into a slot by TMA, read by the lanes (one row each,
// swizzled), the finished rows are written back into the same slot and leave as a TMA tile store.  The loads of a warp's first
// two steps and its bias values are requested before the accumulator is waited for.  (Prefetching the remaining residual tiles
// into L2 as well measured no faster: 16384 x 7168 x 2048 with an fp32 residual 448 us with, 444 us without.  Plain 32-byte
// stores from registers instead of slots and tile stores: 4096 x 7168 x 2048 MXFP8 with silu 64 us against 61 us, with a residual 73
// against 63.  Steps of 16 columns, which halve the code: 79 us.)
//
// The kernels are compiled per activation: all of them in one kernel overflow the instruction caches that the epilogue, scale,
// load and MMA warps share (4096 x 7168 x 2048 MXFP8: no activation 61 -> 56 us, silu 71 -> 61, gelu 89 -> 75; MXFP4 61 -> 52, 68 -> 57,
// 76 -> 67; as the kernels stand 55, 61, 66 and 46, 53, 63).
#pragma once
#include "activation.cuh"
#include "gemm_common.cuh"
#include <type_traits>

namespace b200 {

struct NoEpilogue
{
};
struct alignas(64) FusedParams
{
    CUtensorMap map_res;
    const void* bias; // [N]
    int bias_mode;    // OutMode of the bias' type
    const void* res;  // [M, N]
    long long res_ld;
    int res_mode;
    int res_vec;
    int res_tma;      // residual tiles come through map_res
    uint32_t res_step, out_step; // res_ld and the output's pitch as 32-bit numbers (15 rows of either stay below 2^32 elements)
    int act;
    int out_mode;
    int stream;           // residual and output are larger than L2: their lines leave it first
    uint32_t slot_bytes;  // 32 rows x 32 columns of the wider of residual and output: 2048 or 4096
};

// EPI of the kernels: 0 the plain epilogue, else the activation class (persistent kernel) or 1 (the others)
template <int EPI>
using EpilogueParams = std::conditional_t<EPI == 0, NoEpilogue, FusedParams>;

constexpr int kFusedStep      = 32;
constexpr int kFusedWarps     = 8;
constexpr int kFusedBarBytes  = 16 * kFusedWarps;       // two residual barriers per epilogue warp
constexpr int kFusedBiasBytes = 4 * 128 * kFusedWarps;  // a warp's bias values of one tile (at most 128 columns), fp32

// (plain loads throughout: the residual may be the output itself, and it or the bias may come from the kernel just before, which
// this one may overlap up to its dependency wait - the read-only path is for memory that nothing writes meanwhile)
__device__ __forceinline__ uint32_t load_elem_raw(const void* base, int mode, size_t at)
{
    return mode == OUT_F32 ? static_cast<const uint32_t*>(base)[at] : static_cast<const uint16_t*>(base)[at];
}
__device__ __forceinline__ float raw_to_f32(uint32_t raw, int mode)
{
    return mode == OUT_F32 ? __uint_as_float(raw) : mode == OUT_BF16 ? __uint_as_float(raw << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(raw)));
}
__device__ __forceinline__ float load_elem(const void* base, int mode, size_t at) { return raw_to_f32(load_elem_raw(base, mode, at), mode); }

// v[2i], v[2i + 1] += the two 16-bit values of a word
__device__ __forceinline__ void add16x2(float& a, float& b, uint32_t w, bool f16)
{
    if(f16)
    {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a += f.x;
        b += f.y;
    }
    else
    {
        a += __uint_as_float(w << 16);
        b += __uint_as_float(w & 0xFFFF0000u);
    }
}
// What an epilogue warp needs of the slot path: `seq` counts its steps over all tiles (slot = seq & 1).
struct FusedWarp
{
    uint32_t seq;
    uint32_t slots, rbars;  // shared-memory addresses of the two slots and their barriers
    uint8_t* slots_gen;
    float* bias;            // this warp's bias values of the current tile
    int group;              // 0 or 1: the steps it takes
};

__device__ __forceinline__ void fused_load(const FusedWarp& f, const FusedParams& epi, uint32_t seq, int row0, int col0)
{
    const uint32_t esize = epi.res_mode == OUT_F32 ? 4u : 2u;
    const uint32_t bar   = f.rbars + 8u * (seq & 1);
    mbar_arrive_expect_tx(bar, 32u * kFusedStep * esize);
    if(epi.stream)
        tma_load_2d_hint(f.slots + (seq & 1) * epi.slot_bytes, &epi.map_res, bar, col0 * static_cast<int>(esize), row0, l2_evict_first_policy());
    else
        tma_load_2d(f.slots + (seq & 1) * epi.slot_bytes, &epi.map_res, bar, col0 * static_cast<int>(esize), row0);
}

// Before the accumulator of a tile is waited for.  row0, col0: first row of the warp's 32, first column of the tile.
__device__ __forceinline__ void fused_begin(const FusedWarp& f, const FusedParams& epi, int row0, int col0, int bn, int rows_q, int lane)
{
    const int steps = bn / kFusedStep;
    if(epi.bias != nullptr)
    {
        for(int c = f.group; c < steps; c += 2)
        {
            const int q                            = col0 + c * kFusedStep + lane;
            f.bias[(c >> 1) * kFusedStep + lane] = q < rows_q ? load_elem(epi.bias, epi.bias_mode, q) : 0.f;
        }
    }
    if(epi.res_tma != 0 && lane == 0)
    {
        bulk_wait_group_read<0>(); // the slots' last stores have been read
        uint32_t seq = f.seq;
        for(int c = f.group; c < min(steps, 4); c += 2) // (at most two)
            fused_load(f, epi, seq++, row0, col0 + c * kFusedStep);
    }
    __syncwarp();
}

// One warp's share of a tile.  Returns false when a wait ran out.
template <int EPI, typename Params, typename Release>
__device__ __forceinline__ bool fused_tile(FusedWarp& f, const FusedParams& epi, const Params& prm, const CUtensorMap* map_out, uint32_t tacc, int row0, int col0,
                                           int bn, volatile uint32_t* abort_f, int lane, int uc, Release&& release_acc)
{
    constexpr int STEP = kFusedStep;
    const int steps    = bn / STEP;
    const bool out32   = epi.out_mode == OUT_F32;
    const bool out_f16 = epi.out_mode == OUT_F16;
    if(f.group >= steps)
        release_acc();
    for(int c = f.group; c < steps; c += 2, ++f.seq)
    {
        float v[STEP];
        {
            uint32_t r[STEP];
            tmem_ld_x32(tacc + c * STEP, r);
            tmem_ld_wait();
#pragma unroll
            for(int j = 0; j < STEP; ++j)
                v[j] = __uint_as_float(r[j]);
        }
        if(c + 2 >= steps)
            release_acc(); // every column that this warp reads is in registers now
        const int q_first = col0 + c * STEP;
        if(lane == 0)
        {
            if(epi.res_tma == 0)
                bulk_wait_group_read<1>(); // the store that last used this slot has read it
            else if(c >= 2 && c + 2 < steps)
            {
                // the previous step's store has read its slot: the residual tile of the next step goes there
                bulk_wait_group_read<0>();
                fused_load(f, epi, f.seq + 1, row0, q_first + 2 * STEP);
            }
        }
        if(epi.bias != nullptr)
        {
            const float4* b = reinterpret_cast<const float4*>(f.bias + (c >> 1) * STEP);
#pragma unroll
            for(int j = 0; j < STEP / 4; ++j)
            {
                const float4 t = b[j];
                v[4 * j] += t.x;
                v[4 * j + 1] += t.y;
                v[4 * j + 2] += t.z;
                v[4 * j + 3] += t.w;
            }
        }
        activate<EPI>(v, epi.act);
        __syncwarp();
        uint8_t* slot = f.slots_gen + (f.seq & 1) * epi.slot_bytes;
        // a lane's row: 128 bytes of fp32, or 64 of a 16-bit type, in 16-byte pieces swizzled against bank conflicts
        uint8_t* row128 = slot + lane * 128;
        uint8_t* row64  = slot + lane * 64;
        const int x128 = lane & 7, x64 = (lane >> 1) & 3;
        if(epi.res_tma != 0)
        {
            bool ok = bounded_wait(f.rbars + 8u * (f.seq & 1), (f.seq >> 1) & 1, abort_f, prm.status, ST_TIMEOUT_EPILOGUE, 0x4000 + uc);
            ok      = __all_sync(0xffffffffu, ok);
            if(!ok)
                return false;
            if(epi.res_mode == OUT_F32)
            {
#pragma unroll
                for(int j = 0; j < STEP / 4; ++j)
                {
                    const float4 t = *reinterpret_cast<const float4*>(row128 + ((j ^ x128) * 16));
                    v[4 * j] += t.x;
                    v[4 * j + 1] += t.y;
                    v[4 * j + 2] += t.z;
                    v[4 * j + 3] += t.w;
                }
            }
            else
            {
#pragma unroll
                for(int j = 0; j < STEP / 8; ++j)
                {
                    const uint4 t = *reinterpret_cast<const uint4*>(row64 + ((j ^ x64) * 16));
                    add16x2(v[8 * j], v[8 * j + 1], t.x, epi.res_mode == OUT_F16);
                    add16x2(v[8 * j + 2], v[8 * j + 3], t.y, epi.res_mode == OUT_F16);
                    add16x2(v[8 * j + 4], v[8 * j + 5], t.z, epi.res_mode == OUT_F16);
                    add16x2(v[8 * j + 6], v[8 * j + 7], t.w, epi.res_mode == OUT_F16);
                }
            }
            __syncwarp(); // (types of different sizes: a row of one covers rows of the other)
        }
        if(out32)
        {
#pragma unroll
            for(int j = 0; j < STEP / 4; ++j)
                *reinterpret_cast<float4*>(row128 + ((j ^ x128) * 16)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
        else
        {
#pragma unroll
            for(int j = 0; j < STEP / 8; ++j)
                *reinterpret_cast<uint4*>(row64 + ((j ^ x64) * 16)) = make_uint4(pack_out16x2(v[8 * j], v[8 * j + 1], out_f16), pack_out16x2(v[8 * j + 2], v[8 * j + 3], out_f16),
                                                                                  pack_out16x2(v[8 * j + 4], v[8 * j + 5], out_f16), pack_out16x2(v[8 * j + 6], v[8 * j + 7], out_f16));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if(lane == 0 && row0 < prm.rows_p && q_first < prm.rows_q) // partly outside: the store clips
        {
            if(epi.stream)
                tma_store_2d_hint(map_out, f.slots + (f.seq & 1) * epi.slot_bytes, q_first * (out32 ? 4 : 2), row0, l2_evict_first_policy());
            else
                tma_store_2d(map_out, f.slots + (f.seq & 1) * epi.slot_bytes, q_first * (out32 ? 4 : 2), row0);
        }
        // A group for every step, empty where the step lies outside the output and stores nothing: "all groups but the last" then are
        // the steps before the previous one, so that a slot is never written while the store of its last content still reads it.
        if(lane == 0)
            bulk_commit_group();
    }
    return true;
}

// Outputs or residuals whose rows allow no tile copies, and tiles with the weights on the 128-row slot (few rows, a K split over a
// cluster, or rows that start on odd addresses: there the lanes run along the output's columns and plain accesses coalesce).
// Sixteen columns of the accumulator at a time, alternating between the two warps of a quarter, with the residual of the next
// sixteen under way (the first before the accumulator is waited for).
struct FusedPlain
{
    uint32_t raw[16]; // residual of the group that comes next
};

// Sixteen elements `step` apart, of which `valid` exist.  One test of the type and of the tile's edge for all of them: what this
// epilogue costs is instructions (a test per element: 47 of them a value instead of about 20, and 4096 x 4097 x 1024 with
// gelu_tanh and a residual 79 us).
template <typename T>
__device__ __forceinline__ void load16(uint32_t (&raw)[16], const T* src, uint32_t step, int valid)
{
    if(valid >= 16)
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            raw[j] = src[static_cast<size_t>(j * step)];
    }
    else
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            raw[j] = j < valid ? static_cast<uint32_t>(src[static_cast<size_t>(j) * step]) : 0u;
    }
}
template <typename T, typename Convert>
__device__ __forceinline__ void store16(T* dst, const float (&v)[16], uint32_t step, int valid, Convert&& convert)
{
    if(valid >= 16)
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            dst[static_cast<size_t>(j * step)] = convert(v[j]);
    }
    else
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            if(j < valid)
                dst[static_cast<size_t>(j) * step] = convert(v[j]);
    }
}

// v += sixteen raw values of one type
__device__ __forceinline__ void add_raw16(float (&v)[16], const uint32_t (&raw)[16], int mode)
{
    if(mode == OUT_BF16)
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            v[j] += __uint_as_float(raw[j] << 16);
    }
    else if(mode == OUT_F16)
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            v[j] += raw_to_f32(raw[j], OUT_F16);
    }
    else
    {
#pragma unroll
        for(int j = 0; j < 16; ++j)
            v[j] += __uint_as_float(raw[j]);
    }
}
__device__ __forceinline__ void store_rows16(void* out, int mode, size_t at, const float (&v)[16], uint32_t step, int valid)
{
    if(mode == OUT_F32)
        store16(static_cast<float*>(out) + at, v, step, valid, [](float x) { return x; });
    else if(mode == OUT_BF16)
        store16(static_cast<uint16_t*>(out) + at, v, step, valid, [](float x) { return cvt_out16(x, false); });
    else
        store16(static_cast<uint16_t*>(out) + at, v, step, valid, [](float x) { return cvt_out16(x, true); });
}

template <typename Params>
__device__ __forceinline__ void fused_plain_load(FusedPlain& f, const FusedParams& epi, const Params& prm, int p, int q_first)
{
    if(epi.res == nullptr)
        return;
    const bool transposed = prm.transposed_out != 0;
    const int valid       = p < prm.rows_p ? prm.rows_q - q_first : 0;
    const uint32_t step   = transposed ? epi.res_step : 1u;
    const size_t at       = transposed ? static_cast<size_t>(q_first) * epi.res_ld + p : static_cast<size_t>(p) * epi.res_ld + q_first;
    if(epi.res_mode == OUT_F32)
        load16(f.raw, static_cast<const uint32_t*>(epi.res) + at, step, valid);
    else
        load16(f.raw, static_cast<const uint16_t*>(epi.res) + at, step, valid);
}

// Before the accumulator is waited for: the first group's residual into registers, the rest of this warp's part of the tile into
// L2.  The registers of eight warps hold 8 KB of loads, which at the latency of HBM is 1 TB/s, at that of L2 three times as much.
template <typename Params>
__device__ __forceinline__ void fused_plain_begin(FusedPlain& f, const FusedParams& epi, const Params& prm, int p_warp0, int col0, int bn, int group, int lane)
{
    if(epi.res == nullptr)
        return;
    fused_plain_load(f, epi, prm, p_warp0 + lane, col0 + 16 * group);
    if(prm.transposed_out && p_warp0 < prm.rows_p)
    {
        // lane l: row l % 16 of every other group of 16, starting with the second; both ends of its 32 columns
        const int esize = epi.res_mode == OUT_F32 ? 4 : 2;
        const int last  = min(p_warp0 + 31, prm.rows_p - 1);
        for(int c = group + 2 + 2 * (lane >> 4); c < bn / 16; c += 4)
        {
            const int q = col0 + c * 16 + (lane & 15);
            if(q < prm.rows_q)
            {
                const uint8_t* row = static_cast<const uint8_t*>(epi.res) + static_cast<size_t>(q) * epi.res_ld * esize;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(row + static_cast<size_t>(p_warp0) * esize));
                asm volatile("prefetch.global.L2 [%0];" ::"l"(row + static_cast<size_t>(last) * esize));
            }
        }
    }
}

// red / red_stride: the other K slices' partial sums of this thread's row.
template <int EPI, typename Params, typename Release>
__device__ __forceinline__ bool fused_plain_tile(FusedPlain& f, const FusedParams& epi, const Params& prm, uint32_t tacc, int p, int col0, int bn, int group, int csplit,
                                                 const float* red, size_t red_stride, uint32_t red_bar, volatile uint32_t* abort_f, int uc, Release&& release_acc)
{
    const int groups  = bn / 16;
    const bool row_in = p < prm.rows_p, transposed = prm.transposed_out != 0;
    const float bias_p = (epi.bias != nullptr && transposed && row_in) ? load_elem(epi.bias, epi.bias_mode, p) : 0.f;
    if(group >= groups)
        release_acc();
#pragma unroll 1
    for(int c = group; c < groups; c += 2)
    {
        const int q_first = col0 + c * 16;
        const int valid   = row_in ? prm.rows_q - q_first : 0;
        float v[16];
        {
            uint32_t r[16];
            tmem_ld_x16_at(tacc + c * 16, r);
            tmem_ld_wait();
#pragma unroll
            for(int j = 0; j < 16; ++j)
                v[j] = __uint_as_float(r[j]);
        }
        if(c + 2 >= groups)
            release_acc(); // every column that this warp reads is in registers now
        if(csplit > 1)
        {
            if(c == group)
            {
                bool ok = bounded_wait(red_bar, uc & 1, abort_f, prm.status, ST_TIMEOUT_EPILOGUE, 0x3000 + uc);
                ok      = __all_sync(0xffffffffu, ok);
                if(!ok)
                    return false;
            }
            for(int z = 0; z < csplit - 1; ++z)
            {
                const float4* row = reinterpret_cast<const float4*>(red + z * red_stride + c * 16);
#pragma unroll
                for(int j = 0; j < 16; j += 4)
                {
                    const float4 t = row[j / 4];
                    v[j] += t.x;
                    v[j + 1] += t.y;
                    v[j + 2] += t.z;
                    v[j + 3] += t.w;
                }
            }
        }
        if(epi.bias != nullptr)
        {
            if(transposed)
            {
#pragma unroll
                for(int j = 0; j < 16; ++j)
                    v[j] += bias_p;
            }
            else
            {
#pragma unroll
                for(int j = 0; j < 16; ++j)
                    v[j] += j < valid ? load_elem(epi.bias, epi.bias_mode, q_first + j) : 0.f;
            }
        }
        activate<EPI>(v, epi.act);
        if(epi.res != nullptr)
        {
            add_raw16(v, f.raw, epi.res_mode);
            if(c + 2 < groups)
                fused_plain_load(f, epi, prm, p, q_first + 32);
        }
        const size_t at         = transposed ? static_cast<size_t>(q_first) * prm.ldo + p : static_cast<size_t>(p) * prm.ldo + q_first;
        const uint32_t out_step = transposed ? epi.out_step : 1u;
        store_rows16(prm.out, epi.out_mode, at, v, out_step, valid);
    }
    return true;
}

} // namespace b200
