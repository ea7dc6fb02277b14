// extern "C" entry points of the operators between two GEMMs (block_ops.cuh): argument checks and launches.
#include "../../include/aiter_b200.h"
#include "abi_checks.h"
#include "block_ops.cuh"
#include "launch.h"
#include "norm_stream.cuh"

#include <algorithm>
#include <atomic>
#include <string>
#include <type_traits>

using namespace b200;

// defined in abi.cu: stores the message where aiter_get_last_error() finds it
void aiter_b200_set_last_error(const std::string& msg);

namespace {

template <typename Fn>
int safe_call(Fn&& fn)
{
    try
    {
        aiter_b200_set_last_error(std::string());
        fn();
        return 0;
    }
    catch(const std::exception& e)
    {
        aiter_b200_set_last_error(e.what());
    }
    catch(...)
    {
        aiter_b200_set_last_error("unknown C++ exception");
    }
    return -1;
}

// Makes a device current for a launch and puts the previous one back.
struct DeviceGuard
{
    int prev = 0, cur;
    explicit DeviceGuard(int device) : cur(device)
    {
        B200_CUDA(cudaGetDevice(&prev));
        if(prev != cur)
            B200_CUDA(cudaSetDevice(cur));
    }
    ~DeviceGuard()
    {
        if(prev != cur)
            cudaSetDevice(prev);
    }
};

int float_type(const aiter_tensor_t* t, const char* fn, const char* name)
{
    switch(t->dtype_)
    {
    case AITER_DTYPE_bf16: return OUT_BF16;
    case AITER_DTYPE_fp16: return OUT_F16;
    case AITER_DTYPE_fp32: return OUT_F32;
    default: fail(fn, ": ", name, " must be bf16, fp16 or fp32 (got ", dtype_name(t->dtype_), ")");
    }
}
int bytes_of(int dt) { return dt == OUT_F32 ? 4 : dt == OUT_E2M1 || dt == OUT_MXFP8 ? 1 : 2; }

// every vector of eight elements of every row starts on a 16-byte boundary
bool rows_aligned(const void* p, long long ld, int dt) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * bytes_of(dt)) % 16 == 0; }

// A row of [M, n] values, contiguous along n (`written`: the rows do not overlap one another)
RowTensor row_tensor(const aiter_tensor_t* t, const char* fn, const char* name, long long M, long long n, bool written = false)
{
    require_tensor(t, fn, name, 2);
    B200_CHECK(t->shape[0] == M && t->shape[1] == n, fn, ": ", name, " must be [", M, ", ", n, "] (got [", t->shape[0], ", ", t->shape[1], "])");
    require_rows_contiguous(t, fn, name);
    B200_CHECK(!written || M <= 1 || t->strides[0] >= n, fn, ": the rows of ", name, " overlap one another");
    const int dt = float_type(t, fn, name);
    require_rows(t, bytes_of(dt), fn, name);
    return RowTensor{t->ptr, t->strides[0], dt};
}

// [n] for every row, or [groups, n]: M must be a multiple of groups, row r uses entry r / (M / groups).  `scalar`: [groups, 1] is
// allowed too (one value an entry).
RowParam row_param(const aiter_tensor_t* t, const char* fn, const char* name, long long M, long long n, int* scalar = nullptr)
{
    if(scalar != nullptr)
        *scalar = 0;
    if(t == nullptr)
        return RowParam{nullptr, 0, OUT_BF16, 1u};
    require_tensor(t, fn, name, t->ndim == 1 ? 1 : 2);
    B200_CHECK(t->ptr != nullptr, fn, ": ", name, " has a null data pointer");
    const int dt       = float_type(t, fn, name);
    require_rows(t, bytes_of(dt), fn, name);
    const long long w  = t->shape[t->ndim - 1];
    const bool one     = scalar != nullptr && t->ndim == 2 && w == 1 && n != 1;
    B200_CHECK(w == n || one, fn, ": ", name, " must have ", n, " columns (got ", w, ")");
    if(!one)
        require_rows_contiguous(t, fn, name);
    if(scalar != nullptr)
        *scalar = one;
    if(t->ndim == 1)
        return RowParam{t->ptr, 0, dt, 1u};
    const long long groups = t->shape[0];
    B200_CHECK(groups >= 1 && M % groups == 0, fn, ": ", name, " has ", groups, " entries, which do not divide ", M, " rows");
    return RowParam{t->ptr, groups == 1 ? 0 : t->strides[0], dt, static_cast<unsigned>(M / groups)};
}

Span span(const RowTensor& t, long long rows, long long n)
{
    const int b = bytes_of(t.dt);
    return Span{reinterpret_cast<uintptr_t>(t.ptr), t.ld * b, (t.dt == OUT_E2M1 ? n / 2 : n * b), rows};
}
bool same_rows(const RowTensor& a, const RowTensor& b) { return a.ptr == b.ptr && a.ld == b.ld && a.dt == b.dt; }

// The MX output of [M, n] values: data as fp8 [M, n] or fp4x2 / uint8 [M, n / 2], and its scale array
void mx_output(const aiter_tensor_t* out, const aiter_tensor_t* scales, int layout, const char* fn, long long M, long long n, RowTensor& y, BlockScales& sf)
{
    const bool fp4 = out->dtype_ != AITER_DTYPE_fp8;
    B200_CHECK(n % 32 == 0, fn, ": MX outputs need a multiple of 32 columns (got ", n, ")");
    B200_CHECK(layout >= 0 && layout <= 2, fn, ": shuffle_scale must be 0 (plain), 1 (e8m0_shuffle) or 2 ((m/32,k/4,32,4))");
    B200_CHECK(out->shape[0] == M && out->shape[1] == (fp4 ? n / 2 : n), fn, ": out must be [M, ", (fp4 ? "n/2" : "n"), "]");
    require_rows_contiguous(out, fn, "out");
    B200_CHECK(M <= 1 || out->strides[0] >= out->shape[1], fn, ": the rows of out overlap one another");
    B200_CHECK((reinterpret_cast<uintptr_t>(out->ptr) & 7) == 0 && out->strides[0] % 8 == 0, fn, ": out rows must start on 8-byte boundaries");
    require_tensor(scales, fn, "scales", 2);
    B200_CHECK(scales->dtype_ == AITER_DTYPE_fp8_e8m0 || scales->dtype_ == AITER_DTYPE_u8, fn, ": scales must be e8m0 / uint8 (got ", dtype_name(scales->dtype_), ")");
    require_dense(scales, fn, "scales");
    const long long kb = n / 32, rows32 = (M + 31) / 32 * 32;
    if(layout == QSL_E8M0_SHUFFLE)
        B200_CHECK(scales->shape[0] >= rows32 && scales->shape[1] >= (kb + 7) / 8 * 8 && scales->shape[1] % 8 == 0, fn, ": shuffled scales must be [>= pad32(M), pad8(n/32)]");
    else if(layout == QSL_M32K4)
    {
        B200_CHECK(n % 128 == 0, fn, ": the (m/32,k/4,32,4) scale layout needs n % 128 == 0");
        B200_CHECK(scales->shape[0] >= rows32 && scales->shape[1] == kb, fn, ": scales must be [pad32(M), n/32]");
    }
    else
        B200_CHECK(scales->shape[0] >= M && scales->shape[1] >= kb, fn, ": scales must be [M, n/32]");
    B200_CHECK(layout == QSL_PLAIN || (reinterpret_cast<uintptr_t>(scales->ptr) & 7) == 0, fn, ": scales must be 8-byte aligned");
    y  = RowTensor{out->ptr, out->strides[0], fp4 ? OUT_E2M1 : OUT_MXFP8};
    sf = BlockScales{static_cast<uint8_t*>(scales->ptr), static_cast<int>(scales->shape[1]), layout};
}
bool is_mx(const aiter_tensor_t* out)
{
    return out->dtype_ == AITER_DTYPE_fp8 || out->dtype_ == AITER_DTYPE_fp4x2 || out->dtype_ == AITER_DTYPE_u8;
}

template <typename... Params>
void launch_smem(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, const Params&... prm)
{
    // the set-up of the kernel may run while its predecessor in the stream drains: it waits before its first access
    cudaLaunchConfig_t lc{};
    lc.gridDim  = grid;
    lc.blockDim = block;
    lc.dynamicSmemBytes = smem;
    lc.stream   = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs    = attr;
    lc.numAttrs = programmatic_launch_enabled() ? 1 : 0;
    B200_CUDA(cudaLaunchKernelEx(&lc, kernel, prm...));
    count_launch();
}

template <typename... Params>
void launch(void (*kernel)(Params...), dim3 grid, dim3 block, cudaStream_t stream, const Params&... prm)
{
    launch_smem(kernel, grid, block, 0, stream, prm...);
}
constexpr unsigned kLongRow = 16384; // elements of a row that the register kernels hold at most (512 threads x 4 groups of eight)

template <int CNT, bool SHIFT>
void launch_norm_rows(const NormParams& prm, dim3 grid, dim3 block, cudaStream_t stream)
{
    const bool x32 = prm.x.dt == OUT_F32, r32 = prm.res.ptr != nullptr && prm.res.dt == OUT_F32;
    if(x32 && r32)
        launch(norm_rows_kernel<CNT, true, true, SHIFT>, grid, block, stream, prm);
    else if(x32)
        launch(norm_rows_kernel<CNT, true, false, SHIFT>, grid, block, stream, prm);
    else if(r32)
        launch(norm_rows_kernel<CNT, false, true, SHIFT>, grid, block, stream, prm);
    else
        launch(norm_rows_kernel<CNT, false, false, SHIFT>, grid, block, stream, prm);
}

// ---- many rows: the streaming kernels, for the usual types (types that differ more run the general kernels)
struct StreamShape
{
    unsigned threads;
    unsigned fixed;  // bytes of shared memory besides the rows
    unsigned budget; // bytes an SM's CTAs may use for rows in flight
    bool flat;       // the kernel for rows of any width: a grid that is a multiple of 8
    NormStreamLayout lay;
};

using StreamKernel = void (*)(NormParams, NormStreamLayout);
template <StreamKernel kernel>
bool launch_stream(const NormParams& prm, StreamShape sh, int sms, cudaStream_t stream)
{
    static std::atomic<unsigned long long> attr_done{0}; // a bit per device
    static std::atomic<unsigned> regs{0};
    int dev = 0;
    B200_CUDA(cudaGetDevice(&dev));
    if(dev >= 64 || !((attr_done.load() >> dev) & 1))
    {
        B200_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
        cudaFuncAttributes attr{};
        B200_CUDA(cudaFuncGetAttributes(&attr, kernel));
        regs = static_cast<unsigned>(attr.numRegs);
        if(dev < 64)
            attr_done.fetch_or(1ull << dev);
    }
    // as many CTAs as the registers allow, two to four rows in flight for each
    const unsigned row = sh.lay.x_bytes + sh.lay.r_bytes;
    unsigned ctas      = std::max(1u, std::min({24u, 2048u / sh.threads, 65536u / ((regs + 7) / 8 * 8 * sh.threads)}));
    while(ctas > 1 && (2u * row + sh.fixed) * ctas > 192u * 1024u)
        --ctas;
    const unsigned share = sh.budget / ctas;
    sh.lay.stages        = std::min(4u, std::max(2u, share > sh.fixed ? (share - sh.fixed) / row : 0u));
    if((sh.lay.stages * row + sh.fixed) * ctas > 200u * 1024u)
        return false;
    sh.lay.param_off = sh.lay.stages * row;
    unsigned grid    = std::min(prm.M, static_cast<unsigned>(sms) * ctas);
    if(sh.flat)
    {
        // A CTA brings its parameters to shared memory first: with fewer than four rows for it the general kernel's shifted groups are ahead
        // (us, here and there: 1000 x 1155 10 and 6.3, 400 x 3001 13.5 and 8.4, 1142 x 5287 41 and 26; with 5 to 18 rows 16384 x 301 27 and
        // 31, 8200 x 1155 38 and 40, 8192 x 4097 50 and 76).
        grid = std::max(8u, grid / 8 * 8);
        if(prm.M < 4 * grid)
            return false;
    }
    launch_smem(kernel, dim3(grid), dim3(sh.threads), static_cast<size_t>(sh.lay.stages) * row + sh.fixed, stream, prm, sh.lay);
    return true;
}
template <int XD, int RD, int PD>
bool launch_stream_shape(const NormParams& prm, unsigned cnt, const StreamShape& sh, int sms, cudaStream_t stream)
{
    if(cnt == 0)
    {
        // short rows: 8 warps a CTA, each 4 groups of 32 / lanes rows
        const unsigned lanes = prm.n <= 64 ? 8 : prm.n <= 128 ? 16 : 32;
        const unsigned per   = 8 * 4 * (32 / lanes);
        const dim3 grid((prm.M + per - 1) / per), block(256);
        lanes == 8    ? launch(norm_short_kernel<XD, RD, PD, 8>, grid, block, stream, prm)
        : lanes == 16 ? launch(norm_short_kernel<XD, RD, PD, 16>, grid, block, stream, prm)
                      : launch(norm_short_kernel<XD, RD, PD, 32>, grid, block, stream, prm);
        return true;
    }
    if(sh.flat)
        return cnt == 1 ? launch_stream<norm_stream_flat_kernel<XD, RD, PD, 1>>(prm, sh, sms, stream) : launch_stream<norm_stream_flat_kernel<XD, RD, PD, 2>>(prm, sh, sms, stream);
    if(cnt == 1)
        return launch_stream<norm_stream_kernel<XD, RD, PD, 1, false>>(prm, sh, sms, stream);
    if(cnt == 4)
        return launch_stream<norm_stream_kernel<XD, RD, PD, 4, false>>(prm, sh, sms, stream);
    return prm.n == 16 * sh.threads ? launch_stream<norm_stream_kernel<XD, RD, PD, 2, true>>(prm, sh, sms, stream)
                                    : launch_stream<norm_stream_kernel<XD, RD, PD, 2, false>>(prm, sh, sms, stream);
}

// Whether element 0 of every row has the same place in its group of eight elements in all of x, residual, h and y, with the groups
// aligned to their size
bool same_phase(const NormParams& prm)
{
    auto first = [](const RowTensor& v) { return reinterpret_cast<uintptr_t>(v.ptr) / bytes_of(v.dt); };
    for(const RowTensor* v : {&prm.res, &prm.h, &prm.y})
        if(v->ptr != nullptr && (((first(*v) ^ first(prm.x)) & 7) != 0 || ((v->ld ^ prm.x.ld) & 7) != 0))
            return false;
    return true;
}

// Returns false where the general kernels have to serve the call.
bool try_norm_stream(const NormParams& prm, bool aligned, int device, int sms, cudaStream_t stream)
{
    const unsigned n = prm.n;
    const int xd = prm.x.dt, rd = prm.res.ptr != nullptr ? prm.res.dt : (prm.h.ptr != nullptr ? prm.h.dt : xd);
    // (short rows on any address: the general kernel's shifted groups, 16384 x 203 16 us against 22)
    if(prm.M <= 2u * static_cast<unsigned>(sms) || (!aligned && n < 256) || (prm.h.ptr != nullptr && prm.h.dt != rd))
        return false;
    // one type for all parameters
    int pd          = -1;
    unsigned params = 0;
    for(const RowParam* p : {&prm.weight, &prm.bias, &prm.post_weight, &prm.post_bias, &prm.gate})
    {
        if(p->ptr == nullptr || (p == &prm.gate && prm.gate_scalar))
            continue;
        if(pd >= 0 && pd != p->dt)
            return false;
        pd = p->dt;
        ++params;
    }
    const int half = xd == OUT_F32 ? (rd == OUT_F32 ? OUT_BF16 : rd) : xd; // the call's 16-bit type
    if(pd < 0)
        pd = half;
    if((xd != OUT_F32 && rd != OUT_F32 && xd != rd) || (pd != OUT_F32 && pd != half))
        return false;
    StreamShape sh{};
    unsigned cnt, elems = n;
    const unsigned param_bytes = pd == OUT_F32 ? 4u : 2u;
    if(aligned)
    {
        if(n > kLongRow)
            return false;
        cnt        = n > 8192 ? 4 : n > 512 ? 2 : n > 256 ? 1 : 0; // (0: the short-row kernel)
        sh.threads = cnt == 0 ? 256 : ((n + 8 * cnt - 1) / (8 * cnt) + 31) / 32 * 32;
        // The parameters are read through L1: several vectors of them want 100 KB of the SM's memory left to it (16384 x 8192, rms, with
        // 192 KB of rows in flight and with 128: two norms and a gate 200 us and 184, a weight alone 191 with either.  A weight and a gate
        // without the first norm go the other way, 173 and 194: the rule counts vectors, not norms).
        sh.budget = (params * n * param_bytes > 20u * 1024u ? 128u : 192u) * 1024u;
    }
    else
    {
        // groups of eight elements have to be aligned in every tensor at once
        if(n > 8000 || !same_phase(prm))
            return false;
        elems      = (n + 14) / 8 * 8; // (a row touches at most that many elements in whole groups)
        // two groups a thread, one where whole warps of them would leave more than 15 % of the lanes idle by comparison
        // (8200 x 1155 with per-sample parameters: 192 lanes for 146 groups 41 us, 160 lanes 35; 16384 x 1001, where both fit, 34 and 38)
        auto warps = [&](unsigned c) { return ((elems / 8 + c - 1) / c + 31) / 32; };
        cnt        = n > 512 && 100 * warps(1) > 85 * 2 * warps(2) ? 2 : 1;
        if(warps(cnt) > 16)
            cnt = 2;
        sh.threads = warps(cnt) * 32;
        sh.flat    = true;
        sh.budget  = 192u * 1024u;
        sh.lay.param_pitch = elems * param_bytes;
        sh.fixed           = params * sh.lay.param_pitch;
    }
    sh.lay.x_bytes = elems * bytes_of(xd);
    sh.lay.r_bytes = prm.res.ptr != nullptr ? elems * bytes_of(rd) : 0u;
    sh.lay.report = wait_report(device);
    auto run = [&](auto x, auto r) {
        constexpr int XD = decltype(x)::value, RD = decltype(r)::value, HD = XD != OUT_F32 ? XD : RD != OUT_F32 ? RD : OUT_BF16;
        return pd == OUT_F32 ? launch_stream_shape<XD, RD, OUT_F32>(prm, cnt, sh, sms, stream) : launch_stream_shape<XD, RD, HD>(prm, cnt, sh, sms, stream);
    };
    using B = std::integral_constant<int, OUT_BF16>;
    using H = std::integral_constant<int, OUT_F16>;
    using F = std::integral_constant<int, OUT_F32>;
    if(xd == OUT_BF16)
        return rd == OUT_BF16 ? run(B{}, B{}) : run(B{}, F{});
    if(xd == OUT_F16)
        return rd == OUT_F16 ? run(H{}, H{}) : run(H{}, F{});
    return rd == OUT_BF16 ? run(F{}, B{}) : rd == OUT_F16 ? run(F{}, H{}) : run(F{}, F{});
}

void launch_norm(const NormParams& prm, bool aligned, int device, int sms, cudaStream_t stream)
{
    const unsigned n = prm.n;
    if(try_norm_stream(prm, aligned, device, sms, stream))
        return;
    const unsigned vecs = aligned ? (n + 7) / 8 : (n + 14) / 8; // groups of eight that a row touches at most
    if(vecs > kLongRow / 8)
    {
        if(aligned)
            launch(norm_long_kernel<8>, dim3(prm.M), dim3(512), stream, prm);
        else
            launch(norm_long_kernel<1>, dim3(prm.M), dim3(512), stream, prm);
        return;
    }
    // one group a thread where there are few rows (the shortest chain), up to four where the machine is full
    const bool few     = prm.M <= 2u * static_cast<unsigned>(sms);
    // (SHIFT holds more registers a group: two at most, so that an SM keeps 32 warps, though under the 64 registers of that bound a thread
    // spills 72 to 128 bytes; 4096 x 9001 126 us, four groups a thread took 30 % longer)
    const unsigned cnt = aligned ? (vecs > 1024 ? 4 : few ? 1 : vecs >= 1024 ? 4 : vecs >= 256 ? 2 : 1) : vecs > 1024 || (!few && vecs >= 256) ? 2 : 1;
    unsigned t         = ((vecs + cnt - 1) / cnt + 31) / 32 * 32;
    if(!aligned && vecs <= 16)
        t = vecs <= 8 ? 8 : 16;
    const unsigned r = t <= 32 ? 128 / t : 1; // (short rows: as many as make four warps a CTA)
    const dim3 grid((prm.M + r - 1) / r), block(t, r);
    if(!aligned)
        cnt == 1 ? launch_norm_rows<1, true>(prm, grid, block, stream) : launch_norm_rows<2, true>(prm, grid, block, stream);
    else if(cnt == 1)
        launch_norm_rows<1, false>(prm, grid, block, stream);
    else if(cnt == 2)
        launch_norm_rows<2, false>(prm, grid, block, stream);
    else
        launch_norm_rows<4, false>(prm, grid, block, stream);
}

template <bool X32, int ACT>
void launch_act_mul(ActMulParams& prm, int out_dt, bool aligned, cudaStream_t stream)
{
    const char* big = "act_and_mul: too many elements";
    if(out_dt > OUT_F32)
    {
        const unsigned long long tiles = static_cast<unsigned long long>((prm.M + 31ull) / 32) * ((prm.n / 32 + 7) / 8);
        B200_CHECK(tiles < (1ull << 31), big);
        const dim3 grid(static_cast<unsigned>(tiles)), block(256);
        out_dt == OUT_E2M1 ? launch(act_mul_mx_kernel<X32, true, ACT>, grid, block, stream, prm) : launch(act_mul_mx_kernel<X32, false, ACT>, grid, block, stream, prm);
        return;
    }
    prm.row_vecs                   = aligned ? prm.n / 8 : (prm.n + 14) / 8;
    const unsigned per             = !aligned && X32 ? 256 : 512; // vectors of a CTA
    const unsigned long long ctas  = (static_cast<unsigned long long>(prm.M) * prm.row_vecs + per - 1) / per;
    B200_CHECK(ctas < (1ull << 31), big);
    const dim3 grid(static_cast<unsigned>(ctas)), block(256);
    aligned ? launch(act_mul_kernel<X32, ACT>, grid, block, stream, prm) : launch(act_mul_shift_kernel<X32, ACT>, grid, block, stream, prm);
}

} // namespace

extern "C" int aiter_b200_gated_residual_norm(aiter_tensor_t* out, aiter_tensor_t* scales, aiter_tensor_t* residual_out, aiter_tensor_t* x,
                                              aiter_tensor_t* residual, aiter_tensor_t* weight, aiter_tensor_t* bias, aiter_tensor_t* gate,
                                              aiter_tensor_t* post_weight, aiter_tensor_t* post_bias, float residual_scale,
                                              float weight_offset, float eps, int norm, int post_norm, int shuffle_scale, void* stream)
{
    return safe_call([&] {
        const char* fn = "aiter_b200_gated_residual_norm";
        require_tensor(x, fn, "x", 2);
        require_tensor(out, fn, "out", 2);
        const long long M = x->shape[0], n = x->shape[1];
        B200_CHECK(n > 0, fn, ": x must have at least one column");
        B200_CHECK(M < (1LL << 31) && n < (1LL << 31), fn, ": dimension too large");
        B200_CHECK(norm == 0 || norm == 1, fn, ": norm must be 0 (rms) or 1 (layer), got ", norm);
        B200_CHECK(post_norm != 0 || (post_weight == nullptr && post_bias == nullptr), fn, ": post_weight and post_bias go with the first norm only");
        NormParams prm{};
        prm.x = row_tensor(x, fn, "x", M, n);
        if(residual != nullptr)
            prm.res = row_tensor(residual, fn, "residual", M, n);
        if(residual_out != nullptr)
            prm.h = row_tensor(residual_out, fn, "residual_out", M, n, true);
        prm.weight      = row_param(weight, fn, "weight", M, n);
        prm.bias        = row_param(bias, fn, "bias", M, n);
        prm.gate        = row_param(gate, fn, "gate", M, n, &prm.gate_scalar);
        prm.post_weight = row_param(post_weight, fn, "post_weight", M, n);
        prm.post_bias   = row_param(post_bias, fn, "post_bias", M, n);
        if(is_mx(out))
            mx_output(out, scales, shuffle_scale, fn, M, n, prm.y, prm.sf);
        else
        {
            B200_CHECK(scales == nullptr, fn, ": scales go with an MX output only");
            prm.y = row_tensor(out, fn, "out", M, n, true);
        }
        for(const aiter_tensor_t* t : {out, scales, residual_out, residual, weight, bias, gate, post_weight, post_bias})
            require_same_device(x, t, fn, "an argument");
        if(M == 0)
            return;
        // written rows share no memory with one another or with what other rows read; a tensor may be updated in place
        const Span sx = span(prm.x, M, n), sy = span(prm.y, M, n);
        B200_CHECK((prm.y.dt <= OUT_F32 && same_rows(prm.y, prm.x)) || !overlap(sx, sy), fn, ": out overlaps x");
        if(residual != nullptr)
            B200_CHECK((prm.y.dt <= OUT_F32 && same_rows(prm.y, prm.res)) || !overlap(span(prm.res, M, n), sy), fn, ": out overlaps residual");
        if(residual_out != nullptr)
        {
            const Span sh = span(prm.h, M, n);
            B200_CHECK(!overlap(sh, sy), fn, ": residual_out overlaps out");
            B200_CHECK(same_rows(prm.h, prm.x) || !overlap(sx, sh), fn, ": residual_out overlaps x");
            B200_CHECK(residual == nullptr || same_rows(prm.h, prm.res) || !overlap(span(prm.res, M, n), sh), fn, ": residual_out overlaps residual");
        }
        // every row reads the parameters, and the scales are written beside the rows
        auto span_of = [&](const aiter_tensor_t* t) {
            const int size = t == scales ? 1 : t->dtype_ == AITER_DTYPE_fp32 ? 4 : 2;
            const bool one = t->ndim == 1;
            return Span{reinterpret_cast<uintptr_t>(t->ptr), one ? 0 : t->strides[0] * size, t->shape[t->ndim - 1] * size, one ? 1 : t->shape[0]};
        };
        for(const aiter_tensor_t* t : {weight, bias, gate, post_weight, post_bias, scales})
        {
            if(t == nullptr)
                continue;
            const Span st = span_of(t);
            B200_CHECK(!overlap(st, sy) && (residual_out == nullptr || !overlap(st, span(prm.h, M, n))), fn, ": an output overlaps a parameter or the scales");
            B200_CHECK(t != scales || (!overlap(st, sx) && (residual == nullptr || !overlap(st, span(prm.res, M, n)))), fn, ": scales overlap an input");
            B200_CHECK(t == scales || scales == nullptr || !overlap(st, span_of(scales)), fn, ": scales overlap a parameter");
        }
        prm.post          = post_norm != 0;
        prm.layer         = norm;
        prm.res_scale     = residual_scale;
        prm.weight_offset = weight_offset;
        prm.eps           = eps;
        prm.inv_n         = 1.0f / static_cast<float>(n);
        prm.M             = static_cast<unsigned>(M);
        prm.n             = static_cast<unsigned>(n);
        bool aligned = n % 8 == 0 && rows_aligned(prm.x.ptr, prm.x.ld, prm.x.dt) && (prm.res.ptr == nullptr || rows_aligned(prm.res.ptr, prm.res.ld, prm.res.dt)) &&
                       (prm.h.ptr == nullptr || rows_aligned(prm.h.ptr, prm.h.ld, prm.h.dt)) && (prm.y.dt > OUT_F32 || rows_aligned(prm.y.ptr, prm.y.ld, prm.y.dt));
        for(const RowParam* p : {&prm.weight, &prm.bias, &prm.post_weight, &prm.post_bias})
            aligned = aligned && (p->ptr == nullptr || rows_aligned(p->ptr, p->ld, p->dt));
        aligned = aligned && (prm.gate.ptr == nullptr || prm.gate_scalar || rows_aligned(prm.gate.ptr, prm.gate.ld, prm.gate.dt));
        B200_CHECK(aligned || prm.y.dt <= OUT_F32, fn, ": with an MX output every row of every argument must start on a 16-byte boundary");
        const int sms = device_sm_count(x->device_id);
        DeviceGuard guard(x->device_id);
        launch_norm(prm, aligned, x->device_id, sms, static_cast<cudaStream_t>(stream));
    });
}

extern "C" int aiter_b200_act_and_mul(aiter_tensor_t* out, aiter_tensor_t* scales, aiter_tensor_t* input, int activation, int shuffle_scale, void* stream)
{
    return safe_call([&] {
        const char* fn = "aiter_b200_act_and_mul";
        require_tensor(input, fn, "input", 2);
        require_tensor(out, fn, "out", 2);
        const long long M = input->shape[0], n2 = input->shape[1], n = n2 / 2;
        B200_CHECK(n2 > 0 && n2 % 2 == 0, fn, ": input must have an even number of columns (got ", n2, ")");
        B200_CHECK(M < (1LL << 31) && n2 < (1LL << 31), fn, ": dimension too large");
        B200_CHECK(activation > ACT_NONE && activation < ACT_COUNT, fn, ": activation must be 1 (relu), 2 (silu), 3 (gelu) or 4 (gelu_tanh), got ", activation);
        const RowTensor in = row_tensor(input, fn, "input", M, n2);
        RowTensor y{};
        ActMulParams prm{};
        if(is_mx(out))
            mx_output(out, scales, shuffle_scale, fn, M, n, y, prm.sf);
        else
        {
            B200_CHECK(scales == nullptr, fn, ": scales go with an MX output only");
            y = row_tensor(out, fn, "out", M, n, true);
        }
        require_same_device(input, out, fn, "out");
        require_same_device(input, scales, fn, "scales");
        if(M == 0)
            return;
        B200_CHECK((y.dt <= OUT_F32 && same_rows(y, in)) || !overlap(span(in, M, n2), span(y, M, n)), fn, ": out overlaps the input (only the gate half may be overwritten in place)");
        if(scales != nullptr)
        {
            const Span st{reinterpret_cast<uintptr_t>(scales->ptr), scales->strides[0], scales->shape[1], scales->shape[0]};
            B200_CHECK(!overlap(st, span(in, M, n2)) && !overlap(st, span(y, M, n)), fn, ": scales overlap the input or out");
        }
        prm.in     = in.ptr;
        prm.in_ld  = in.ld;
        prm.in_dt  = in.dt;
        prm.out    = y.ptr;
        prm.out_ld = y.ld;
        prm.out_dt = y.dt;
        prm.act    = activation;
        prm.M      = static_cast<unsigned>(M);
        prm.n      = static_cast<unsigned>(n);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        const bool in_vec    = n % 8 == 0 && rows_aligned(in.ptr, in.ld, in.dt);
        const bool x32       = in.dt == OUT_F32;
        B200_CHECK(in_vec || y.dt <= OUT_F32, fn, ": with an MX output the input's rows must start on 16-byte boundaries");
        DeviceGuard guard(input->device_id);
        const bool aligned = in_vec && (y.dt > OUT_F32 || rows_aligned(y.ptr, y.ld, y.dt));
        auto go = [&](auto act) {
            constexpr int ACT = decltype(act)::value;
            x32 ? launch_act_mul<true, ACT>(prm, y.dt, aligned, s) : launch_act_mul<false, ACT>(prm, y.dt, aligned, s);
        };
        switch(activation)
        {
        case ACT_RELU: return go(std::integral_constant<int, ACT_RELU>{});
        case ACT_SILU: return go(std::integral_constant<int, ACT_SILU>{});
        case ACT_GELU: return go(std::integral_constant<int, ACT_GELU>{});
        default: return go(std::integral_constant<int, ACT_GELU_TANH>{});
        }
    });
}
