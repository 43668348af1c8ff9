// attend.cu — kvops_attend_hot: attention of drafted tokens over the hot rows that their top-K
// lists name and over one another's drafted rows along a tree (the formulas are in
// include/kvops_b200.h).
//
// One CTA per query row: its keys in chunks of 128, the scores of a chunk by warps, then the
// running maximum and sum of the softmax and the weighted sum of the rows' first 512 values, all in
// fp32. Every query row reads its keys again, so the rows come from L2 heads * tokens times.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <string>

#include "kvops_internal.cuh"
#include "quant.cuh"

namespace kvb {
namespace {

constexpr int kValueDim = 512;            // values of a row that the output sums
constexpr int kKeyDim = 576;              // values of a row that the scores use
constexpr uint32_t kStoredBytes = 656;    // of a stored row of 512 + 64 values
constexpr int kThreads = 128;
constexpr int kChunk = 128;               // keys per chunk

// Values 2j and 2j + 1 of a row: 16-bit, or read back from its stored form.
template <typename T, typename Code>
__device__ __forceinline__ float2 stored_pair(const uint8_t *row, int j)
{
    if (j >= kValueDim / 2) return T::unpack(*reinterpret_cast<const uint32_t *>(row + kValueDim + 16 + 4 * (j - 256)));
    const float scale = *reinterpret_cast<const float *>(row + kValueDim + j / 64 * 4);
    const float4 c = Code::decode4(*reinterpret_cast<const uint16_t *>(row + 2 * j));
    return T::unpack(T::pack(__fmul_rn(c.x, scale), __fmul_rn(c.y, scale)));
}

template <typename T, typename Code, bool kStored>
__device__ __forceinline__ float2 key_pair(const uint8_t *row, int j, bool draft)
{
    if (kStored && !draft) return stored_pair<T, Code>(row, j);
    return T::unpack(*reinterpret_cast<const uint32_t *>(row + 4 * j));
}

template <typename T, typename Code, bool kStored>
__global__ void __launch_bounds__(kThreads) attend_kernel(const KvopsAttend a)
{
    __shared__ const uint8_t *s_key[kChunk];  // nullptr: no key
    __shared__ float s_p[kChunk];
    __shared__ float2 s_q[kKeyDim / 2];
    __shared__ float s_red[4];
    const uint32_t h = blockIdx.x % a.heads, t = blockIdx.x / a.heads % a.tokens, r = blockIdx.x / a.heads / a.tokens;
    if (static_cast<int32_t>(r) >= *reinterpret_cast<const int32_t *>(a.num_real)) return;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint8_t *q = reinterpret_cast<const uint8_t *>(a.q) +
                       2 * (r * a.q_stride_req + t * a.q_stride_token + h * a.q_stride_head);
    for (int j = threadIdx.x; j < kKeyDim / 2; j += kThreads) s_q[j] = T::unpack(*reinterpret_cast<const uint32_t *>(q + 4 * j));
    const uint64_t row_bytes = kStored ? kStoredBytes : 2 * kKeyDim;
    const int64_t req = a.top_k > 0 ? reinterpret_cast<const int64_t *>(a.req_pool_indices)[r] : -1;
    const bool in_pool = req >= 0 && req < static_cast<int64_t>(a.pool_size);
    const uint8_t *hot = reinterpret_cast<const uint8_t *>(a.hot_row_base) + (in_pool ? req * a.hot_req_stride_rows * row_bytes : 0);
    const int32_t *slots = reinterpret_cast<const int32_t *>(a.topk_device_slots) + r * a.slots_stride_req + t * a.slots_stride_token;
    const uint64_t word = a.tree != 0 ? reinterpret_cast<const uint64_t *>(a.tree)[r * a.tokens + t] : (2ull << t) - 1;
    float top = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    const uint32_t total = a.top_k + a.drafts;
    for (uint32_t base = 0; base < total; base += kChunk) {
        __syncthreads();
        const uint32_t k = base + threadIdx.x;
        const uint8_t *key = nullptr;
        if (k < a.top_k) {
            const int32_t slot = slots[k];
            if (in_pool && slot >= 0 && static_cast<uint32_t>(slot) < a.hot_rows) key = hot + slot * row_bytes;
        } else if (k < total) {
            const uint32_t j = k - a.top_k;
            if ((word >> j) & 1)
                key = reinterpret_cast<const uint8_t *>(a.draft_rows) + 2 * (r * a.draft_stride_req + j * a.draft_stride_row);
        }
        s_key[threadIdx.x] = key;
        __syncthreads();
        for (int i = warp; i < kChunk; i += 4) {
            float s = -INFINITY;
            const uint8_t *row = s_key[i];
            if (row != nullptr) {
                const bool draft = base + i >= a.top_k;
                float d = 0.f;
                for (int j = lane; j < kKeyDim / 2; j += 32) {
                    const float2 x = key_pair<T, Code, kStored>(row, j, draft), y = s_q[j];
                    d += x.x * y.x + x.y * y.y;
                }
                for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
                s = d * a.scale;
            }
            if (lane == 0) s_p[i] = s;
        }
        __syncthreads();
        float m = s_p[threadIdx.x];
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if (lane == 0) s_red[warp] = m;
        __syncthreads();
        const float was = top;
        for (int w = 0; w < 4; ++w) top = fmaxf(top, s_red[w]);
        const float ref = top == -INFINITY ? 0.f : top;
        const float back = expf(was - ref);
        const float p = s_key[threadIdx.x] != nullptr ? expf(s_p[threadIdx.x] - ref) : 0.f;
        __syncthreads();
        s_p[threadIdx.x] = p;
        __syncthreads();
        sum *= back;
        for (int i = 0; i < 4; ++i) acc[i] *= back;
        for (int i = 0; i < kChunk; ++i) {
            const uint8_t *row = s_key[i];
            if (row == nullptr) continue;
            const float w = s_p[i];
            sum += w;
            const bool draft = base + i >= a.top_k;
            const float2 x = key_pair<T, Code, kStored>(row, 2 * threadIdx.x, draft);
            const float2 y = key_pair<T, Code, kStored>(row, 2 * threadIdx.x + 1, draft);
            acc[0] += w * x.x;
            acc[1] += w * x.y;
            acc[2] += w * y.x;
            acc[3] += w * y.y;
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 v;
    v.x = T::pack(acc[0] * inv, acc[1] * inv);
    v.y = T::pack(acc[2] * inv, acc[3] * inv);
    reinterpret_cast<uint2 *>(a.out)[static_cast<uint64_t>(blockIdx.x) * (kValueDim / 4) + threadIdx.x] = v;
    if (a.lse != 0 && threadIdx.x == 0)
        reinterpret_cast<float *>(a.lse)[blockIdx.x] = sum == 0.f ? -INFINITY : logf(sum) + (top == -INFINITY ? 0.f : top);
}

int invalid(const char *msg) { return set_last_error(KVOPS_E_INVALID, msg); }

// The argument checks that both entry points share.
int check_shape(const KvopsAttend *a)
{
    if (!is_inited()) return set_last_error(KVOPS_E_NOT_INITED, "kvops not inited");
    if (a == nullptr) return invalid("attend_hot: the arguments are NULL");
    if (a->tokens == 0 || a->tokens > 64) return invalid("attend_hot: tokens must be in [1, 64]");
    if (a->heads == 0 || a->heads > 128) return invalid("attend_hot: heads must be in [1, 128]");
    if (a->drafts > 64) return invalid("attend_hot: drafts must be <= 64");
    if (a->top_k > (1u << 24) || a->max_num_reqs > (1u << 16))
        return invalid("attend_hot: top_k / max_num_reqs out of range");
    if (a->row_format > KVOPS_ROW_INT8) return invalid("attend_hot: row_format must be 0, 1 or 2");
    if (a->row_dtype > KVOPS_DTYPE_BF16) return invalid("attend_hot: row_dtype must be 0 or 1");
    return KVOPS_OK;
}

template <typename T>
cudaError_t launch_as(const KvopsAttend &a, cudaStream_t s)
{
    const uint32_t grid = a.max_num_reqs * a.tokens * a.heads;
    switch (a.row_format) {
        case KVOPS_ROW_E4M3: attend_kernel<T, E4m3, true><<<grid, kThreads, 0, s>>>(a); break;
        case KVOPS_ROW_INT8: attend_kernel<T, Int8, true><<<grid, kThreads, 0, s>>>(a); break;
        default: attend_kernel<T, Int8, false><<<grid, kThreads, 0, s>>>(a); break;
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace kvb

extern "C" int kvops_attend_workspace(const KvopsAttend *a, uint64_t *out_bytes)
{
    const int rc = kvb::check_shape(a);
    if (rc != KVOPS_OK) return rc;
    if (out_bytes == nullptr) return kvb::invalid("attend_workspace: out_bytes is NULL");
    *out_bytes = 0;
    return KVOPS_OK;
}

extern "C" int kvops_attend_hot(const KvopsAttend *a, uint64_t stream)
{
    using kvb::invalid;
    int rc = kvb::check_shape(a);
    if (rc != KVOPS_OK) return rc;
    if (a->max_num_reqs == 0) return KVOPS_OK;
    if (a->q == 0 || a->out == 0 || a->num_real == 0) return invalid("attend_hot: a tensor address is 0");
    if (a->top_k > 0 && (a->hot_row_base == 0 || a->req_pool_indices == 0 || a->topk_device_slots == 0))
        return invalid("attend_hot: a tensor address is 0");
    if (a->drafts > 0 && a->draft_rows == 0) return invalid("attend_hot: a tensor address is 0");
    if ((a->q | a->out | a->workspace | (a->top_k > 0 ? a->hot_row_base : 0) | (a->drafts > 0 ? a->draft_rows : 0)) % 16 != 0)
        return invalid("attend_hot: q, out, hot rows, draft rows and workspace must be 16-byte aligned");
    if ((a->q_stride_req | a->q_stride_token | a->q_stride_head) % 8 != 0 ||
        (a->drafts > 0 && (a->draft_stride_req | a->draft_stride_row) % 8 != 0))
        return invalid("attend_hot: strides of q and draft rows must be multiples of 8 values");
    if (a->lse % 4 != 0 || a->num_real % 4 != 0 || a->topk_device_slots % 4 != 0 || a->req_pool_indices % 8 != 0 ||
        a->tree % 8 != 0)
        return invalid("attend_hot: lse, num_real, slots, pool indices and tree must have their types' alignment");
    uint64_t need = 0;
    rc = kvops_attend_workspace(a, &need);
    if (rc != KVOPS_OK) return rc;
    if (need > 0 && (a->workspace == 0 || a->workspace_bytes < need))
        return invalid("attend_hot: the workspace is smaller than kvops_attend_workspace says");
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = a->row_dtype == KVOPS_DTYPE_FP16 ? kvb::launch_as<kvb::Fp16>(*a, s)
                                                           : kvb::launch_as<kvb::Bf16>(*a, s);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return kvb::set_last_error(KVOPS_E_CUDA, (std::string("launch attend_hot: ") + cudaGetErrorString(e)).c_str());
    }
    return KVOPS_OK;
}
