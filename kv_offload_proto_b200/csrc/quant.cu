// quant.cu — the row copies of rows.cu between 16-bit rows and 8-bit stored rows (quant.cuh):
// kvops_export_quant_alllayer and kvops_export_quant quantise rows as they are written to their
// segments, kvops_import_quant reads the miss rows back into 16-bit hot rows.
//
// A 1152-byte row and its 656 stored bytes cross memory once, whichever way: the bound is HBM (or
// the link to the segment).
// Writing, a warp takes a tile of positions, one per lane, lists the rows it found in shared memory, and
// takes them as one flat array of groups of 128 values: 16 units of 16 bytes, one for each lane of a
// half-warp, which takes eight groups at a time, so that values are read once, from registers to codes.
// No two warps wait for each other. 8192 rows of 61 layers, 903 MB: 188 us, 4.8 TB/s. The instructions
// were 63% of the issue slots with an address for each group; hence four groups to an address.
// Reading, a CTA takes a tile, as rows.cu does, since few positions may be misses, and 16 codes (32
// bytes) a thread at a time. 262,144 of 524,288 positions, 479 MB: 132 us, 3.6 TB/s (123 to 135 on different
// GPUs); copying as many rows of these sizes from and to random places, without any rule or arithmetic, takes
// 98 us. Neither a warp a tile (136 us) nor the next tile's positions loaded ahead (136 us) came nearer to it.
#include <stdint.h>

#include "kvops_internal.cuh"
#include "quant.cuh"
#include "rows_common.cuh"

namespace kvb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;  // 16-byte units in flight per thread

// i / d for the unit indexes of a tile: multiply-high with ceil(2^32 / d), exact while the
// product of index and divisor is below 2^32 (host-checked), else a division (magic 0).
__device__ __forceinline__ uint32_t div_magic(uint32_t i, uint32_t d, uint32_t magic)
{
    return magic ? __umulhi(i, magic) : i / d;
}

// The multipliers for a row's groups (writing) or units of 16 codes (reading), and for its plain units.
struct Magics {
    uint32_t quant, plain;
};

// The rows that a group of kGroup threads (a warp, or the CTA) takes: src[i] -> dst[i].
template <int kGroup>
struct List {
    const uint8_t *src[kGroup];
    uint8_t *dst[kGroup];
};

// Lists the accepted rows of the lanes; returns how many.
__device__ __forceinline__ int list_rows(List<32> &list, bool ok, const uint8_t *src, uint8_t *dst, int lane)
{
    const unsigned mask = __ballot_sync(0xFFFFFFFFu, ok);
    const int at = __popc(mask & ((1u << lane) - 1u));
    __syncwarp();  // the rows listed before have been read
    if (ok) {
        list.src[at] = src;
        list.dst[at] = dst;
    }
    __syncwarp();
    return __popc(mask);
}

// Copies the rows' plain parts, `units` of 16 bytes each.
template <int kGroup>
__device__ __forceinline__ void copy_plain(const List<kGroup> &list, int n, uint32_t units, uint32_t magic,
                                           uint32_t src_at, uint32_t dst_at, int thread)
{
    const uint32_t total = n * units;
    for (uint32_t i0 = thread; i0 < total; i0 += kGroup * kUnroll) {
        uint4 v[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = i0 + k * kGroup, row = div_magic(i, units, magic);
            if (i < total) v[k] = load_stream(reinterpret_cast<const uint4 *>(list.src[row] + src_at) + (i - row * units));
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = i0 + k * kGroup, row = div_magic(i, units, magic);
            if (i < total) reinterpret_cast<uint4 *>(list.dst[row] + dst_at)[i - row * units] = v[k];
        }
    }
}

// Quantises n listed 16-bit rows into stored rows. kRun groups of a row share its addresses.
template <typename T, typename Code, int kRun>
__device__ __forceinline__ void encode_rows(const RowCodec &c, const List<32> &list, int n, Magics m, int lane)
{
    copy_plain<32>(list, n, c.plain_elems / 8, m.plain, 2 * c.quant_elems, c.quant_elems + codec_scale_bytes(c), lane);
    const uint32_t per_row = c.quant_elems / (kQuantGroup * kRun), total = static_cast<uint32_t>(n) * per_row;  // runs
    constexpr int kRuns = 8 / kRun;
    const int half = lane >> 4, unit = lane & 15;
    for (uint32_t r0 = 0; r0 < total; r0 += 2 * kRuns) {
        const uint32_t mine = r0 + half * kRuns;
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < kRuns; ++j) {
            const uint32_t row = div_magic(mine + j, per_row, m.quant), run = mine + j - row * per_row;
            const bool any = mine + j < total;
            const uint4 *at = any ? reinterpret_cast<const uint4 *>(list.src[row]) + run * (16 * kRun) + unit : nullptr;
#pragma unroll
            for (int k = 0; k < kRun; ++k) {
                v[j * kRun + k] = make_uint4(0u, 0u, 0u, 0u);
                if (any) v[j * kRun + k] = load_stream(at + 16 * k);
            }
        }
        uint2 codes[8];
        float scale;
        encode_groups<T, Code>(v, unit, codes, &scale);
#pragma unroll
        for (int j = 0; j < kRuns; ++j) {
            const uint32_t row = div_magic(mine + j, per_row, m.quant), run = mine + j - row * per_row;
            if (mine + j < total) {
                uint2 *at = reinterpret_cast<uint2 *>(list.dst[row]) + run * (16 * kRun) + unit;
#pragma unroll
                for (int k = 0; k < kRun; ++k) at[16 * k] = codes[j * kRun + k];
            }
        }
        const uint32_t own = mine + scale_group(unit) / kRun;  // the run of the group whose scale this lane has
        if (own < total && (unit & 1) == 0) {
            const uint32_t row = div_magic(own, per_row, m.quant);
            const uint32_t group = (own - row * per_row) * kRun + scale_group(unit) % kRun;
            float *scales = reinterpret_cast<float *>(list.dst[row] + c.quant_elems);
            scales[group] = scale;
            if (kRun == 1 && group + 1 == per_row)  // the padding, as zeros (no run of four leaves any)
                for (uint32_t g = per_row; g < codec_scale_bytes(c) / 4; ++g) scales[g] = 0.f;
        }
    }
}

// Reads n listed stored rows back into 16-bit rows, with the whole CTA.
template <typename T, typename Code>
__device__ __forceinline__ void decode_rows(const RowCodec &c, const List<kThreads> &list, int n, Magics m)
{
    const uint32_t units = c.quant_elems / 16, total = static_cast<uint32_t>(n) * units;  // (eight to a group)
    for (uint32_t i0 = threadIdx.x; i0 < total; i0 += kThreads * kUnroll) {
        uint4 v[kUnroll];
        float scale[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = i0 + k * kThreads, row = div_magic(i, units, m.quant), unit = i - row * units;
            if (i < total) {
                const uint8_t *s = list.src[row];
                v[k] = load_stream(reinterpret_cast<const uint4 *>(s) + unit);
                scale[k] = *reinterpret_cast<const volatile float *>(s + c.quant_elems + unit / 8 * 4);
            }
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const uint32_t i = i0 + k * kThreads, row = div_magic(i, units, m.quant), unit = i - row * units;
            if (i < total) {
                uint4 *d = reinterpret_cast<uint4 *>(list.dst[row]) + 2 * unit;
                d[0] = decode_unit<T, Code>(make_uint2(v[k].x, v[k].y), scale[k]);
                d[1] = decode_unit<T, Code>(make_uint2(v[k].z, v[k].w), scale[k]);
            }
        }
    }
    copy_plain<kThreads>(list, n, c.plain_elems / 8, m.plain, c.quant_elems + codec_scale_bytes(c), 2 * c.quant_elems,
                         threadIdx.x);
}

// The number of positions of the launch's real batch rows. Launched as programmatic dependents, like
// gather_kernel (rows.cu): wait for the kernel before (the SIEVE step) to end before its outputs are read.
__device__ __forceinline__ int64_t real_positions(const GatherParams &p)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int32_t num_real = p.num_real != nullptr ? *p.num_real : 0;
    if (num_real > static_cast<int32_t>(p.max_num_reqs)) num_real = static_cast<int32_t>(p.max_num_reqs);
    return num_real > 0 ? static_cast<int64_t>(num_real) * p.top_k : 0;
}

// The rule for one position: its segment row and hot row.
__device__ __forceinline__ bool rows_of(const GatherParams &p, const RowCodec &c, int64_t pos, const uint8_t **seg_row,
                                        uint8_t **hot_row)
{
    if (p.is_miss[pos] == 0) return false;
    const int64_t bid = pos / p.top_k;
    const int32_t slot = p.slots[pos];
    const int64_t req = p.req_pool[bid];
    if (!gather_source(p, pos, 1, p.topk[pos], slot, req, p.host_base[bid], seg_row)) return false;
    *hot_row = p.hot + static_cast<uint64_t>(req) * p.hot_req_stride_bytes +
               static_cast<uint64_t>(slot) * codec_row_bytes(c);
    return true;
}

// Miss rows read back under the gather's rules.
template <typename T, typename Code>
__global__ void __launch_bounds__(kThreads, 4) import_quant_kernel(const GatherParams p, const RowCodec c, int tile,
                                                                   Magics magics)
{
    __shared__ List<kThreads> list;
    __shared__ int s_n;
    const int thread = threadIdx.x;
    const int64_t total = real_positions(p), step = static_cast<int64_t>(gridDim.x) * tile;
    if (thread == 0) s_n = 0;
    __syncthreads();
    for (int64_t pos = static_cast<int64_t>(blockIdx.x) * tile + thread; pos - thread < total; pos += step) {
        const uint8_t *seg_row = nullptr;
        uint8_t *hot_row = nullptr;
        const bool ok = thread < tile && pos < total && rows_of(p, c, pos, &seg_row, &hot_row);
        list_append(ok, seg_row, hot_row, list.src, list.dst, &s_n);
        __syncthreads();
        decode_rows<T, Code>(c, list, s_n, magics);
        __syncthreads();
        if (thread == 0) s_n = 0;
        __syncthreads();
    }
    __syncthreads();
    if (thread == 0) arrive_and_publish(p.st);
}

// Flagged hot rows written under the gather's rules.
template <typename T, typename Code, int kRun>
__global__ void __launch_bounds__(kThreads, 4) scatter_quant_kernel(const GatherParams p, const RowCodec c, int tile,
                                                                    Magics magics)
{
    __shared__ List<32> lists[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // (tiles of a CTA's warps lie a grid apart, so that few positions use many CTAs)
    const int64_t total = real_positions(p), step = static_cast<int64_t>(gridDim.x) * kWarps * tile;
    for (int64_t pos = (static_cast<int64_t>(warp) * gridDim.x + blockIdx.x) * tile + lane; pos - lane < total; pos += step) {
        const uint8_t *seg_row = nullptr;
        uint8_t *hot_row = nullptr;
        const bool ok = lane < tile && pos < total && rows_of(p, c, pos, &seg_row, &hot_row);
        const int n = list_rows(lists[warp], ok, hot_row, const_cast<uint8_t *>(seg_row), lane);
        encode_rows<T, Code, kRun>(c, lists[warp], n, magics, lane);
    }
    __syncthreads();
    if (threadIdx.x == 0) arrive_and_publish(p.st);
}

template <typename T, typename Code, int kRun>
__global__ void __launch_bounds__(kThreads, 4) export_quant_kernel(const ExportQuantParams p, int tile, Magics magics)
{
    __shared__ List<32> lists[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t total = p.units_per_layer * p.layer_num;
    for (uint64_t base = (static_cast<uint64_t>(warp) * gridDim.x + blockIdx.x) * tile; base < total;
         base += static_cast<uint64_t>(gridDim.x) * kWarps * tile) {
        const uint64_t u = base + lane;
        bool ok = false;
        const uint8_t *src = nullptr;
        uint8_t *dst = nullptr;
        if (lane < tile && u < total) {
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
        const int n = list_rows(lists[warp], ok, src, dst, lane);
        encode_rows<T, Code, kRun>(p.codec, lists[warp], n, magics, lane);
    }
    __syncthreads();
    if (threadIdx.x == 0) arrive_and_publish(p.st);
}

// Positions per tile and grid of a launch.
struct Shape {
    int tile, grid;
};

Shape shape_of(uint64_t positions, int sm_count, bool write)
{
    Shape s;
    const uint64_t ctas = static_cast<uint64_t>(sm_count > 0 ? sm_count : 148) * 4;
    if (write) {
        // At least eight tiles a warp, so that the last one costs little (8192 rows of 61 layers: 189 us, with
        // 32 positions a tile 215), down to tiles of four rows, which are one round of loads; below that,
        // one tile a warp.
        s.tile = 32;
        while (s.tile > 4 && positions <= 8 * ctas * kWarps * (s.tile / 2)) s.tile /= 2;
        while (s.tile > 1 && positions <= ctas * kWarps * (s.tile / 2)) s.tile /= 2;
    } else {
        // One for every thread, since few may be misses; fewer where that leaves CTAs without any (131,072
        // positions, a fifth of them misses: 19 us, with 64 positions a tile 25).
        s.tile = kThreads;
        while (s.tile > 16 && positions <= ctas * (s.tile / 2)) s.tile /= 2;
    }
    const uint64_t tiles = (positions + s.tile - 1) / s.tile;
    s.grid = static_cast<int>(tiles < 1 ? 1 : (tiles < ctas ? tiles : ctas));
    return s;
}

// The multiplier of div_magic for indexes up to one round past a tile's last, or 0.
uint32_t magic_of(uint64_t d)
{
    return d != 0 && d * (kThreads * d + kThreads * kUnroll) < (1ull << 32) ? static_cast<uint32_t>(((1ull << 32) + d - 1) / d) : 0u;
}

// Four groups of a row at a time, where the row has that many.
bool by_fours(const RowCodec &c) { return c.quant_elems % (4 * kQuantGroup) == 0; }

Magics magics_of(const RowCodec &c, bool write)
{
    return {magic_of(!write ? c.quant_elems / 16 : c.quant_elems / (by_fours(c) ? 4 * kQuantGroup : kQuantGroup)),
            magic_of(c.plain_elems / 8)};
}

template <typename T, typename Code>
cudaError_t launch_gather_as(const GatherParams &p, const RowCodec &c, bool write, cudaStream_t s, int sm_count)
{
    const Shape sh = shape_of(static_cast<uint64_t>(p.max_num_reqs) * p.top_k, sm_count, write);
    const Magics magics = magics_of(c, write);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sh.grid);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!write) return cudaLaunchKernelEx(&cfg, import_quant_kernel<T, Code>, p, c, sh.tile, magics);
    return by_fours(c) ? cudaLaunchKernelEx(&cfg, scatter_quant_kernel<T, Code, 4>, p, c, sh.tile, magics)
                       : cudaLaunchKernelEx(&cfg, scatter_quant_kernel<T, Code, 1>, p, c, sh.tile, magics);
}

template <typename T, typename Code>
cudaError_t launch_export_as(const ExportQuantParams &p, cudaStream_t s, int sm_count)
{
    const Shape sh = shape_of(p.units_per_layer * p.layer_num, sm_count, true);
    const Magics magics = magics_of(p.codec, true);
    if (by_fours(p.codec)) export_quant_kernel<T, Code, 4><<<sh.grid, kThreads, 0, s>>>(p, sh.tile, magics);
    else export_quant_kernel<T, Code, 1><<<sh.grid, kThreads, 0, s>>>(p, sh.tile, magics);
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
