// quant.cu — the row copies of rows.cu between 16-bit rows and 8-bit stored rows (quant.cuh):
// kvops_export_quant_alllayer and kvops_export_quant quantise rows as they are written to their
// segments, kvops_import_quant reads the miss rows back into 16-bit hot rows.
//
// A 1152-byte row and its 656 stored bytes cross memory once, whichever way: the bound is HBM (or
// the link to the segment). A CTA evaluates a tile of positions, one per thread, into a shared
// list as rows.cu does, and then takes the listed rows as one flat array of 16-byte units of
// eight values. A group of 128 values is 16 units, so it always lies in the 16 lanes of a
// half-warp, whose maximum four shuffles give: the values are read once, from registers to codes.
#include <stdint.h>

#include "kvops_internal.cuh"
#include "quant.cuh"
#include "rows_common.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // units in flight per thread

// i / d for the unit indexes of a tile: multiply-high with ceil(2^32 / d), exact while the
// product of index and divisor is below 2^32 (host-checked), else a division (magic 0).
__device__ __forceinline__ uint32_t div_magic(uint32_t i, uint32_t d, uint32_t magic)
{
    return magic ? __umulhi(i, magic) : i / d;
}

// Copies the 16-byte units [0, units) of n rows (src[i] + src_off -> dst[i] + dst_off).
__device__ __forceinline__ void cta_copy_plain(const uint8_t *const *src, uint8_t *const *dst, int n, uint32_t units,
                                               uint32_t src_off, uint32_t dst_off)
{
    const uint32_t total = static_cast<uint32_t>(n) * units;
    for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
        const uint32_t r = i / units, u = i - r * units;
        const uint4 v = load_stream(reinterpret_cast<const uint4 *>(src[r] + src_off) + u);
        reinterpret_cast<uint4 *>(dst[r] + dst_off)[u] = v;
    }
}

// Quantises n 16-bit rows src[i] into the stored rows dst[i]. Every thread of the CTA calls it.
template <typename T, typename Code>
__device__ __forceinline__ void cta_encode_rows(const RowCodec &c, const uint8_t *const *src, uint8_t *const *dst,
                                                int n, uint32_t magic)
{
    const uint32_t units = c.quant_elems / 8;
    const uint32_t total = static_cast<uint32_t>(n) * units;
    const uint32_t rounds = (total + kThreads * kUnroll - 1) / (kThreads * kUnroll);
    for (uint32_t it = 0; it < rounds; ++it) {
        uint4 v[kUnroll];
        uint32_t row[kUnroll], unit[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = (it * kUnroll + k) * kThreads + threadIdx.x;
            row[k] = div_magic(i, units, magic);
            unit[k] = i - row[k] * units;
            v[k] = make_uint4(0u, 0u, 0u, 0u);
            if (i < total) v[k] = load_stream(reinterpret_cast<const uint4 *>(src[row[k]]) + unit[k]);
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            // total is a multiple of 16: a half-warp's lanes are all inside or all outside, and
            // every lane takes part in the shuffles.
            float scale;
            const uint2 codes = encode_unit<T, Code>(v[k], &scale);
            if ((it * kUnroll + k) * kThreads + threadIdx.x < total) {
                uint8_t *d = dst[row[k]];
                reinterpret_cast<uint2 *>(d)[unit[k]] = codes;
                if ((unit[k] & 15u) == 0) {
                    float *scales = reinterpret_cast<float *>(d + c.quant_elems);
                    scales[unit[k] / 16] = scale;
                    if (unit[k] + 16 == units)  // the padding, as zeros
                        for (uint32_t g = units / 16; g < codec_scale_bytes(c) / 4; ++g) scales[g] = 0.f;
                }
            }
        }
    }
    cta_copy_plain(src, dst, n, c.plain_elems / 8, 2 * c.quant_elems, c.quant_elems + codec_scale_bytes(c));
}

// Reads n stored rows src[i] back into the 16-bit rows dst[i].
template <typename T, typename Code>
__device__ __forceinline__ void cta_decode_rows(const RowCodec &c, const uint8_t *const *src, uint8_t *const *dst,
                                                int n, uint32_t magic)
{
    const uint32_t units = c.quant_elems / 8;
    const uint32_t total = static_cast<uint32_t>(n) * units;
    for (uint32_t i0 = threadIdx.x; i0 < total; i0 += kThreads * kUnroll) {
        uint2 v[kUnroll];
        float scale[kUnroll];
        uint32_t row[kUnroll], unit[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = i0 + k * kThreads;
            row[k] = div_magic(i, units, magic);
            unit[k] = i - row[k] * units;
            if (i < total) {
                const uint8_t *s = src[row[k]];
                v[k] = load_stream(reinterpret_cast<const uint2 *>(s) + unit[k]);
                scale[k] = *reinterpret_cast<const volatile float *>(s + c.quant_elems + unit[k] / 16 * 4);
            }
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            if (i0 + k * kThreads < total)
                reinterpret_cast<uint4 *>(dst[row[k]])[unit[k]] = decode_unit<T, Code>(v[k], scale[k]);
        }
    }
    cta_copy_plain(src, dst, n, c.plain_elems / 8, c.quant_elems + codec_scale_bytes(c), 2 * c.quant_elems);
}

// Miss rows read back (kWrite false) or flagged hot rows written (true) under the gather's rules.
template <typename T, typename Code, bool kWrite>
__global__ void __launch_bounds__(kThreads, 4) gather_quant_kernel(const GatherParams p, const RowCodec c,
                                                                   uint32_t tile, uint32_t magic)
{
    __shared__ const uint8_t *s_src[kThreads];
    __shared__ uint8_t *s_dst[kThreads];
    __shared__ int s_n;
    // Launched as a programmatic dependent, like gather_kernel (rows.cu): wait for the kernel
    // before (the SIEVE step) to end before its outputs are read.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    int32_t num_real = p.num_real != nullptr ? *p.num_real : 0;
    if (num_real > static_cast<int32_t>(p.max_num_reqs)) num_real = static_cast<int32_t>(p.max_num_reqs);
    const int64_t total = num_real > 0 ? static_cast<int64_t>(num_real) * p.top_k : 0;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * tile; base < total;
         base += static_cast<int64_t>(gridDim.x) * tile) {
        const int64_t pos = base + threadIdx.x;
        const uint8_t *seg_row = nullptr;
        uint8_t *hot_row = nullptr;
        bool ok = false;
        if (threadIdx.x < tile && pos < total && p.is_miss[pos] != 0) {
            const int64_t bid = pos / p.top_k;
            const int32_t slot = p.slots[pos];
            const int64_t req = p.req_pool[bid];
            ok = gather_source(p, pos, 1, p.topk[pos], slot, req, p.host_base[bid], &seg_row);
            if (ok)
                hot_row = p.hot + static_cast<uint64_t>(req) * p.hot_req_stride_bytes +
                          static_cast<uint64_t>(slot) * codec_row_bytes(c);
        }
        list_append(ok, kWrite ? hot_row : seg_row, kWrite ? const_cast<uint8_t *>(seg_row) : hot_row, s_src, s_dst,
                    &s_n);
        __syncthreads();
        if (kWrite) cta_encode_rows<T, Code>(c, s_src, s_dst, s_n, magic);
        else cta_decode_rows<T, Code>(c, s_src, s_dst, s_n, magic);
        __syncthreads();
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
    }
    __syncthreads();
    if (threadIdx.x == 0) arrive_and_publish(p.st);
}

template <typename T, typename Code>
__global__ void __launch_bounds__(kThreads, 4) export_quant_kernel(const ExportParams p, const RowCodec c,
                                                                   uint32_t tile, uint32_t magic)
{
    __shared__ const uint8_t *s_src[kThreads];
    __shared__ uint8_t *s_dst[kThreads];
    __shared__ int s_n;
    const uint64_t total = p.units_per_layer * p.layer_num;
    if (p.seg_null && blockIdx.x == 0 && threadIdx.x == 0) record_error(p.st, KVOPS_ERR_SEG_NULL);
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * tile; base < total;
         base += static_cast<uint64_t>(gridDim.x) * tile) {
        const uint64_t u = base + threadIdx.x;
        bool ok = false;
        const uint8_t *src = nullptr;
        uint8_t *dst = nullptr;
        if (threadIdx.x < tile && u < total) {
            const uint64_t l = u / p.units_per_layer;
            const uint64_t k = u - l * p.units_per_layer;
            uint32_t src_row, seg_row;
            if (export_unit(p, k, &src_row, &seg_row)) {
                if (seg_row >= p.plsr) {
                    const uint64_t idx = l * p.row_cnt + (src_row - p.row_lo);
                    record_error(p.st, KVOPS_ERR_ROW_BASE + static_cast<uint32_t>(idx & 0xFFu) + (1u << 16));
                } else {
                    src = p.src0 + l * p.src_layer_stride + static_cast<uint64_t>(src_row) * codec_row_bytes(c);
                    dst = p.seg + (l * p.plsr + seg_row) * static_cast<uint64_t>(p.row_bytes);
                    ok = true;
                }
            }
        }
        list_append(ok, src, dst, s_src, s_dst, &s_n);
        __syncthreads();
        cta_encode_rows<T, Code>(c, s_src, s_dst, s_n, magic);
        __syncthreads();
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
    }
    __syncthreads();
    if (threadIdx.x == 0) arrive_and_publish(p.st);
}

// Positions per tile (at most one per thread), grid and division constant of a launch.
struct Shape {
    uint32_t tile, magic;
    int grid;
};

Shape shape_of(uint64_t positions, const RowCodec &c, int sm_count)
{
    Shape s;
    const uint64_t cap = static_cast<uint64_t>(sm_count > 0 ? sm_count : 148) * 4;
    s.tile = kThreads;
    while (s.tile > 32 && positions < cap * s.tile * 4) s.tile /= 2;
    const uint64_t tiles = (positions + s.tile - 1) / s.tile;
    s.grid = static_cast<int>(tiles < 1 ? 1 : (tiles < cap ? tiles : cap));
    const uint64_t units = c.quant_elems / 8;
    // indexes run up to one round past the last unit of a tile
    s.magic = units * (s.tile * units + kThreads * kUnroll) < (1ull << 32)
                  ? static_cast<uint32_t>(((1ull << 32) + units - 1) / units) : 0u;
    return s;
}

template <typename T, typename Code>
cudaError_t launch_gather_as(const GatherParams &p, const RowCodec &c, bool write, cudaStream_t s, int sm_count)
{
    const Shape sh = shape_of(static_cast<uint64_t>(p.max_num_reqs) * p.top_k, c, sm_count);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sh.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return write ? cudaLaunchKernelEx(&cfg, gather_quant_kernel<T, Code, true>, p, c, sh.tile, sh.magic)
                 : cudaLaunchKernelEx(&cfg, gather_quant_kernel<T, Code, false>, p, c, sh.tile, sh.magic);
}

template <typename T, typename Code>
cudaError_t launch_export_as(const ExportParams &p, const RowCodec &c, cudaStream_t s, int sm_count)
{
    const Shape sh = shape_of(p.units_per_layer * p.layer_num, c, sm_count);
    export_quant_kernel<T, Code><<<sh.grid, kThreads, 0, s>>>(p, c, sh.tile, sh.magic);
    return cudaGetLastError();
}

cudaError_t launch_gather_any(const GatherParams &p, const RowCodec &c, bool write, cudaStream_t s, int sm_count)
{
    const bool e4m3 = c.format == KVOPS_ROW_E4M3;
    if (c.dtype == KVOPS_DTYPE_FP16)
        return e4m3 ? launch_gather_as<Fp16, E4m3>(p, c, write, s, sm_count)
                    : launch_gather_as<Fp16, Int8>(p, c, write, s, sm_count);
    return e4m3 ? launch_gather_as<Bf16, E4m3>(p, c, write, s, sm_count)
                : launch_gather_as<Bf16, Int8>(p, c, write, s, sm_count);
}

}  // namespace

cudaError_t launch_gather_quant(const GatherParams &p, const RowCodec &c, cudaStream_t s, int sm_count)
{
    return launch_gather_any(p, c, false, s, sm_count);
}

cudaError_t launch_scatter_quant(const GatherParams &p, const RowCodec &c, cudaStream_t s, int sm_count)
{
    return launch_gather_any(p, c, true, s, sm_count);
}

cudaError_t launch_export_quant(const ExportParams &p, const RowCodec &c, cudaStream_t s, int sm_count)
{
    const bool e4m3 = c.format == KVOPS_ROW_E4M3;
    if (c.dtype == KVOPS_DTYPE_FP16)
        return e4m3 ? launch_export_as<Fp16, E4m3>(p, c, s, sm_count) : launch_export_as<Fp16, Int8>(p, c, s, sm_count);
    return e4m3 ? launch_export_as<Bf16, E4m3>(p, c, s, sm_count) : launch_export_as<Bf16, Int8>(p, c, s, sm_count);
}

}  // namespace kvb
