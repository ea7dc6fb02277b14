// Fused GEMM epilogue: out = act(A B^T + bias) + residual on the fp32 accumulator, rounded once.
//
// Row-major output tiles (activations on the 128-row slot) leave in steps of 64 columns (32 where a 32-bit type is
// involved).  Every epilogue warp owns two slots in shared memory: the residual's tile of a step is loaded into a slot by
// TMA, read by the lanes (one row each, 128-byte swizzle), the finished row is written back into the same slot and leaves
// as a TMA tile store.  The loads of a tile's first two steps are issued before the accumulator is waited for and the
// remaining steps are prefetched into L2, so with a second accumulator the residual costs its bytes and no latency.
#pragma once
#include "activation.cuh"
#include "gemm_common.cuh"

namespace b200 {

template <int EPI>
struct EpilogueParams
{
};
template <>
struct alignas(64) EpilogueParams<1>
{
    CUtensorMap map_res;
    const void* bias; // [N]
    int bias_mode;    // OutMode of the bias' type
    int bias_vec;     // 16-byte loads of 8 (4 for fp32) consecutive values are aligned
    const void* res;  // [M, N]
    long long res_ld;
    int res_mode;
    int res_vec;
    int res_tma;      // residual tiles come through map_res
    int act;
    int out_mode;
    int step;             // columns per step of the slot path
    uint32_t slot_bytes;  // 4096, or 8192 where residual and output differ in size (the output then has the upper half)
    uint32_t out_off;
};

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
// v[0 .. N) += N consecutive elements from `at`, of which `valid` exist.
template <int N>
__device__ __forceinline__ void add_row(float (&v)[N], const void* base, int mode, size_t at, int valid, bool vec)
{
    if(vec && valid >= N)
    {
        if(mode == OUT_F32)
        {
#pragma unroll
            for(int i = 0; i < N; i += 4)
            {
                const float4 t = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at + i);
                v[i] += t.x;
                v[i + 1] += t.y;
                v[i + 2] += t.z;
                v[i + 3] += t.w;
            }
        }
        else
        {
#pragma unroll
            for(int i = 0; i < N; i += 8)
            {
                const uint4 t = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + at + i);
                add16x2(v[i], v[i + 1], t.x, mode == OUT_F16);
                add16x2(v[i + 2], v[i + 3], t.y, mode == OUT_F16);
                add16x2(v[i + 4], v[i + 5], t.z, mode == OUT_F16);
                add16x2(v[i + 6], v[i + 7], t.w, mode == OUT_F16);
            }
        }
    }
    else
    {
#pragma unroll
        for(int i = 0; i < N; ++i)
            if(i < valid)
                v[i] += mode == OUT_F32 ? static_cast<const float*>(base)[at + i] : raw_to_f32(static_cast<const uint16_t*>(base)[at + i], mode);
    }
}

// A warp's position in its ring: the number of steps done so far over all tiles (slot = seq & 1).
struct FusedStore
{
    uint32_t seq = 0;
};

__device__ __forceinline__ uint32_t epi_s_fused(uint32_t smem_base, uint32_t epi_off, int w, const EpilogueParams<1>& epi)
{
    return smem_base + epi_off + static_cast<uint32_t>(w) * 2u * epi.slot_bytes;
}

// residual bytes of one step: 32 rows of step columns
__device__ __forceinline__ uint32_t fused_res_bytes(const EpilogueParams<1>& epi) { return 32u * static_cast<uint32_t>(epi.step) * (epi.res_mode == OUT_F32 ? 4u : 2u); }

__device__ __forceinline__ void fused_load(const EpilogueParams<1>& epi, uint32_t seq, int row0, int col0, uint32_t slots, uint32_t rbars)
{
    const uint32_t bar = rbars + 8u * (seq & 1);
    mbar_arrive_expect_tx(bar, fused_res_bytes(epi));
    tma_load_2d(slots + (seq & 1) * epi.slot_bytes, &epi.map_res, bar, col0 * (epi.res_mode == OUT_F32 ? 4 : 2), row0);
}

// Before the accumulator of a tile is waited for: its first two residual tiles are requested (the slots' previous stores have
// been read by then) and the others brought into L2.
__device__ __forceinline__ void fused_begin(const FusedStore& f, const EpilogueParams<1>& epi, int row0, int col0, int bn, uint32_t slots, uint32_t rbars, int lane)
{
    if(epi.res_tma == 0 || lane != 0)
        return;
    bulk_wait_group_read<0>();
    const int steps = bn / epi.step;
    fused_load(epi, f.seq, row0, col0, slots, rbars);
    if(steps > 1)
        fused_load(epi, f.seq + 1, row0, col0 + epi.step, slots, rbars);
    for(int i = 2; i < steps; ++i)
        tma_prefetch_l2_2d(&epi.map_res, (col0 + i * epi.step) * (epi.res_mode == OUT_F32 ? 4 : 2), row0);
}

// One warp's 32 rows of a tile.  row0 / col0: first row and column of the warp's part.  Returns false when a wait ran out.
template <int STEP, typename Params, typename Release>
__device__ __forceinline__ bool fused_tile(FusedStore& f, const EpilogueParams<1>& epi, const Params& prm, const CUtensorMap* map_out, uint32_t tacc, int row0, int col0,
                                           int bn, uint32_t slots, uint8_t* slots_gen, uint32_t rbars, volatile uint32_t* abort_f, int lane, int uc, Release&& release_acc)
{
    const int steps      = bn / STEP;
    const bool out32     = epi.out_mode == OUT_F32;
    const bool out_f16   = epi.out_mode == OUT_F16;
    const int out_esize  = out32 ? 4 : 2;
    for(int c = 0; c < steps; ++c, ++f.seq)
    {
        float v[STEP];
        {
            uint32_t r[STEP];
            if constexpr(STEP == 64)
                tmem_ld_x64(tacc + c * 64, r);
            else
                tmem_ld_x32(tacc + c * 32, r);
            tmem_ld_wait();
#pragma unroll
            for(int j = 0; j < STEP; ++j)
                v[j] = __uint_as_float(r[j]);
        }
        if(c == steps - 1)
            release_acc(); // every column of this accumulator is in registers now
        const int q_first = col0 + c * STEP;
        if(lane == 0)
        {
            if(epi.res_tma == 0)
                bulk_wait_group_read<1>(); // the store that last used this slot has read it
            else if(c > 0 && c + 1 < steps)
            {
                // the previous step's store has read its slot: the residual tile of the next step goes there
                bulk_wait_group_read<0>();
                fused_load(epi, f.seq + 1, row0, q_first + STEP, slots, rbars);
            }
        }
        if(epi.bias != nullptr)
            add_row<STEP>(v, epi.bias, epi.bias_mode, q_first, prm.rows_q - q_first, epi.bias_vec != 0);
        activate(v, epi.act);
        __syncwarp();
        const uint32_t off = (f.seq & 1) * epi.slot_bytes;
        if(epi.res_tma != 0)
        {
            bool ok = bounded_wait(rbars + 8u * (f.seq & 1), (f.seq >> 1) & 1, abort_f, prm.status, ST_TIMEOUT_EPILOGUE, 0x4000 + uc);
            ok      = __all_sync(0xffffffffu, ok);
            if(!ok)
                return false;
            const uint8_t* tile = slots_gen + off;
            if(epi.res_mode == OUT_F32)
            {
                // 32 floats = 128 bytes a row (STEP is 32 whenever a 32-bit type is involved)
#pragma unroll
                for(int j = 0; j < STEP / 4; ++j)
                {
                    const float4 t = *reinterpret_cast<const float4*>(tile + lane * 128 + ((j ^ (lane & 7)) * 16));
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
                    const uint32_t at = STEP == 64 ? lane * 128 + ((j ^ (lane & 7)) * 16) : lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16);
                    const uint4 t     = *reinterpret_cast<const uint4*>(tile + at);
                    add16x2(v[8 * j], v[8 * j + 1], t.x, epi.res_mode == OUT_F16);
                    add16x2(v[8 * j + 2], v[8 * j + 3], t.y, epi.res_mode == OUT_F16);
                    add16x2(v[8 * j + 4], v[8 * j + 5], t.z, epi.res_mode == OUT_F16);
                    add16x2(v[8 * j + 6], v[8 * j + 7], t.w, epi.res_mode == OUT_F16);
                }
            }
        }
        // a lane overwrites only the row it has read; rows of different lanes do not overlap in either type
        uint8_t* dst = slots_gen + off + epi.out_off;
        if(out32)
        {
#pragma unroll
            for(int j = 0; j < STEP / 4; ++j)
                *reinterpret_cast<float4*>(dst + lane * 128 + ((j ^ (lane & 7)) * 16)) = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
        else
        {
#pragma unroll
            for(int j = 0; j < STEP / 8; ++j)
            {
                const uint32_t at = STEP == 64 ? lane * 128 + ((j ^ (lane & 7)) * 16) : lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16);
                *reinterpret_cast<uint4*>(dst + at) = make_uint4(pack_out16x2(v[8 * j], v[8 * j + 1], out_f16), pack_out16x2(v[8 * j + 2], v[8 * j + 3], out_f16),
                                                                 pack_out16x2(v[8 * j + 4], v[8 * j + 5], out_f16), pack_out16x2(v[8 * j + 6], v[8 * j + 7], out_f16));
            }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if(lane == 0 && row0 < prm.rows_p && q_first < prm.rows_q) // partly outside: the store clips
        {
            tma_store_2d(map_out, slots + off + epi.out_off, q_first * out_esize, row0);
            bulk_commit_group();
        }
    }
    return true;
}

} // namespace b200
