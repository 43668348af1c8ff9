// quant.cu — the row copies of rows.cu between 16-bit rows and 8-bit stored rows (quant.cuh):
// kvops_export_quant_alllayer and kvops_export_quant quantise rows as they are written to their
// segments, kvops_import_quant reads the miss rows back into 16-bit hot rows.
//
// A 1152-byte row and its 656 stored bytes cross memory once, whichever way: the bound is HBM (or
// the link to the segment). A CTA evaluates a tile of positions, one per thread, into a shared
// list as rows.cu does, and then takes the listed rows as one flat array of groups of 128 values. A
// group is 16 units of 16 bytes, one for each lane of a half-warp, which takes eight groups at a
// time: the values are read once, from registers to codes.
#include <stdint.h>

#include "kvops_internal.cuh"
#include "quant.cuh"
#include "rows_common.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // 16-code units in flight per thread, reading

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

// Quantises n 16-bit rows src[i] into the stored rows dst[i]. Every thread of the CTA calls it. magic:
// of the groups per row.
template <typename T, typename Code>
__device__ __forceinline__ void cta_encode_rows(const RowCodec &c, const uint8_t *const *src, uint8_t *const *dst,
                                                int n, uint32_t magic)
{
    const uint32_t per_row = c.quant_elems / kQuantGroup, total = static_cast<uint32_t>(n) * per_row;
    const int lane = threadIdx.x & 15;
    for (uint32_t g0 = threadIdx.x / 32 * 16; g0 < total; g0 += kThreads / 16 * 8) {  // (uniform over the warp)
        const uint32_t mine = g0 + (threadIdx.x >> 4 & 1) * 8;
        uint4 v[8];
        uint32_t row[8], group[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            row[k] = div_magic(mine + k, per_row, magic);
            group[k] = mine + k - row[k] * per_row;
            v[k] = make_uint4(0u, 0u, 0u, 0u);
            if (mine + k < total) v[k] = load_stream(reinterpret_cast<const uint4 *>(src[row[k]]) + group[k] * 16 + lane);
        }
        uint2 codes[8];
        float scale;
        encode_groups<T, Code>(v, lane, codes, &scale);
        uint8_t *at = nullptr;  // this lane's group's scale
        uint32_t at_group = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (mine + k >= total) continue;
            uint8_t *d = dst[row[k]];
            reinterpret_cast<uint2 *>(d)[group[k] * 16 + lane] = codes[k];
            if (scale_group(lane) == k && (lane & 1) == 0) {
                at = d + c.quant_elems;
                at_group = group[k];
            }
        }
        if (at != nullptr) {
            reinterpret_cast<float *>(at)[at_group] = scale;
            if (at_group + 1 == per_row)  // the padding, as zeros
                for (uint32_t g = per_row; g < codec_scale_bytes(c) / 4; ++g) reinterpret_cast<float *>(at)[g] = 0.f;
        }
    }
    cta_copy_plain(src, dst, n, c.plain_elems / 8, 2 * c.quant_elems, c.quant_elems + codec_scale_bytes(c));
}

// Reads n stored rows src[i] back into the 16-bit rows dst[i].
template <typename T, typename Code>
__device__ __forceinline__ void cta_decode_rows(const RowCodec &c, const uint8_t *const *src, uint8_t *const *dst,
                                                int n, uint32_t magic)
{
    // units of 16 codes, eight to a group
    const uint32_t units = c.quant_elems / 16;
    const uint32_t total = static_cast<uint32_t>(n) * units;
    for (uint32_t i0 = threadIdx.x; i0 < total; i0 += kThreads * kUnroll) {
        uint4 v[kUnroll];
        float scale[kUnroll];
        uint32_t row[kUnroll], unit[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = i0 + k * kThreads;
            row[k] = div_magic(i, units, magic);
            unit[k] = i - row[k] * units;
            if (i < total) {
                const uint8_t *s = src[row[k]];
                v[k] = load_stream(reinterpret_cast<const uint4 *>(s) + unit[k]);
                scale[k] = *reinterpret_cast<const volatile float *>(s + c.quant_elems + unit[k] / 8 * 4);
            }
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            if (i0 + k * kThreads < total) {
                uint4 *d = reinterpret_cast<uint4 *>(dst[row[k]]) + 2 * unit[k];
                d[0] = decode_unit<T, Code>(make_uint2(v[k].x, v[k].y), scale[k]);
                d[1] = decode_unit<T, Code>(make_uint2(v[k].z, v[k].w), scale[k]);
            }
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
__global__ void __launch_bounds__(kThreads, 4) export_quant_kernel(const ExportQuantParams p, uint32_t tile, uint32_t magic)
{
    __shared__ const uint8_t *s_src[kThreads];
    __shared__ uint8_t *s_dst[kThreads];
    __shared__ int s_n;
    const uint64_t total = p.units_per_layer * p.layer_num;
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * tile; base < total;
         base += static_cast<uint64_t>(gridDim.x) * tile) {
        const uint64_t u = base + threadIdx.x;
        bool ok = false;
        const uint8_t *src = nullptr;
        uint8_t *dst = nullptr;
        if (threadIdx.x < tile && u < total) {
            const uint64_t l = u / p.units_per_layer, k = u - l * p.units_per_layer;
            // Unit k is the k-th row, or (reference map) the last row in range of the k-th stripe, the
            // one that the reference's ascending per-row writes leave in the shared segment row.
            uint64_t row = p.row_lo + k;
            if (p.stripe > 0 && !p.injective) {
                const uint64_t end = (p.row_lo / p.stripe + k + 1) * p.stripe, hi = static_cast<uint64_t>(p.row_lo) + p.row_cnt;
                row = (end < hi ? end : hi) - 1;
            }
            const uint32_t r = static_cast<uint32_t>(row);
            const uint32_t node = node_of(r, p.stripe, p.nodes), seg_row = seg_row_of(r, p.stripe, p.nodes, p.injective != 0);
            if (p.seg[node] == nullptr) {
                record_error(p.st, KVOPS_ERR_SEG_NULL);
            } else if (seg_row >= p.plsr) {
                record_error(p.st, KVOPS_ERR_ROW_BASE + static_cast<uint32_t>((l * p.row_cnt + (row - p.row_lo)) & 0xFFu) +
                                       (1u << 16));
            } else {
                src = p.src0 + l * p.src_layer_stride + row * codec_row_bytes(p.codec);
                dst = p.seg[node] + (l * p.plsr + seg_row) * static_cast<uint64_t>(codec_stored_bytes(p.codec));
                ok = true;
            }
        }
        list_append(ok, src, dst, s_src, s_dst, &s_n);
        __syncthreads();
        cta_encode_rows<T, Code>(p.codec, s_src, s_dst, s_n, magic);
        __syncthreads();
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
    }
    __syncthreads();
    if (threadIdx.x == 0) arrive_and_publish(p.st);
}

// Positions per tile (at most one per thread) and grid of a launch: tiles of `most` positions, or smaller
// ones where those leave CTAs without any.
struct Shape {
    uint32_t tile;
    int grid;
};

Shape shape_of(uint64_t positions, uint32_t most, int sm_count)
{
    Shape s;
    const uint64_t cap = static_cast<uint64_t>(sm_count > 0 ? sm_count : 148) * 4;
    s.tile = most;
    while (s.tile > 16 && positions <= cap * (s.tile / 2)) s.tile /= 2;
    const uint64_t tiles = (positions + s.tile - 1) / s.tile;
    s.grid = static_cast<int>(tiles < 1 ? 1 : (tiles < cap ? tiles : cap));
    return s;
}

// The multiplier of div_magic for indexes up to one round past a tile's last, or 0.
uint32_t magic_of(uint64_t d)
{
    return d * (kThreads * d + kThreads * 8) < (1ull << 32) ? static_cast<uint32_t>(((1ull << 32) + d - 1) / d) : 0u;
}

template <typename T, typename Code>
cudaError_t launch_gather_as(const GatherParams &p, const RowCodec &c, bool write, cudaStream_t s, int sm_count)
{
    const Shape sh = shape_of(static_cast<uint64_t>(p.max_num_reqs) * p.top_k, kThreads, sm_count);
    const uint32_t magic = magic_of(write ? c.quant_elems / kQuantGroup : c.quant_elems / 16);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sh.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return write ? cudaLaunchKernelEx(&cfg, gather_quant_kernel<T, Code, true>, p, c, sh.tile, magic)
                 : cudaLaunchKernelEx(&cfg, gather_quant_kernel<T, Code, false>, p, c, sh.tile, magic);
}

template <typename T, typename Code>
cudaError_t launch_export_as(const ExportQuantParams &p, cudaStream_t s, int sm_count)
{
    const Shape sh = shape_of(p.units_per_layer * p.layer_num, kThreads / 2, sm_count);
    export_quant_kernel<T, Code><<<sh.grid, kThreads, 0, s>>>(p, sh.tile, magic_of(p.codec.quant_elems / kQuantGroup));
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

cudaError_t launch_export_quant(const ExportQuantParams &p, cudaStream_t s, int sm_count)
{
    const bool e4m3 = p.codec.format == KVOPS_ROW_E4M3;
    if (p.codec.dtype == KVOPS_DTYPE_FP16)
        return e4m3 ? launch_export_as<Fp16, E4m3>(p, s, sm_count) : launch_export_as<Fp16, Int8>(p, s, sm_count);
    return e4m3 ? launch_export_as<Bf16, E4m3>(p, s, sm_count) : launch_export_as<Bf16, Int8>(p, s, sm_count);
}

}  // namespace kvb
