// lora.cu -- low-rank adapters of many requests at once
// (include/loom_cuda.h, loom_cuda_lora):
//
//   out[r] = base[r] + scale_a * B_a (A_a x[r]),  a = ids[r]
//
// A row with no adapter (ids[r] outside 0 .. n_adapters - 1) keeps its base.
#include "../../include/loom_cuda.h"
#include "serve.cuh"

namespace loom {
namespace {

struct LoraArgs {
    const float *x, *scales, *base;
    const void *a, *b;
    const int32_t *ranks, *ids;
    float *out, *t;
    int64_t x_stride, base_stride, out_stride, a_row, a_adapter, b_row, b_adapter;
    int n_rows, n_in, n_out, n_adapters, max_rank;
};

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int id) {
    return id < 0 || id >= a.n_adapters ? 0 : min(max(a.ranks[id], 0), a.max_rank);
}

// t[r][k] = scale_a * (A_a x[r])[k], one warp per k
template <class T> __global__ void __launch_bounds__(256) k_lora_shrink(LoraArgs a) {
    const int r = blockIdx.x, lane = threadIdx.x & 31, id = a.ids[r], rank = lora_rank(a, id);
    for (int k = threadIdx.x >> 5; k < rank; k += 8) {
        const T *w = static_cast<const T *>(a.a) + id * a.a_adapter + k * a.a_row;
        const float *x = a.x + r * a.x_stride;
        float s = 0.0f;
        for (int i = lane; i < a.n_in; i += 32) s = fmaf(to_f32(w[i]), x[i], s);
        s = warp_sum(s);
        if (lane == 0) a.t[(size_t)r * a.max_rank + k] = s * a.scales[id];
    }
}

// out[r][o] = base[r][o] + sum_k B_a[o][k] t[r][k], one thread per o
template <class T> __global__ void __launch_bounds__(256) k_lora_expand(LoraArgs a) {
    const int r = blockIdx.x, o = blockIdx.y * 256 + threadIdx.x, id = a.ids[r], rank = lora_rank(a, id);
    if (o >= a.n_out) return;
    const float *t = a.t + (size_t)r * a.max_rank;
    float s = 0.0f;
    for (int k = 0; k < rank; k++) s = fmaf(to_f32(static_cast<const T *>(a.b)[id * a.b_adapter + o * a.b_row + k]), t[k], s);
    a.out[r * a.out_stride + o] = (a.base ? a.base[r * a.base_stride + o] : 0.0f) + s;
}

const char *check(const loom_lora_desc *d) {
    if (!d) return "lora: no descriptor";
    if (!elem_bytes(d->type)) return "lora: type must be LOOM_F32, LOOM_F16 or LOOM_BF16";
    if (!d->n_in || !d->n_out || d->n_in > (1u << 24) || d->n_out > (1u << 24)) return "lora: widths must be 1..2^24";
    if (d->n_rows > (1u << 24)) return "lora: at most 2^24 rows";
    if (d->n_adapters > (1u << 20)) return "lora: at most 2^20 adapters";
    if (d->max_rank > 1024) return "lora: max_rank must be at most 1024";
    return nullptr;
}

size_t ws_bytes_of(const loom_lora_desc *d) { return d->n_rows * d->max_rank * sizeof(float); }

template <class T> cudaError_t launch(const LoraArgs &a, cudaStream_t st) {
    k_lora_shrink<T><<<a.n_rows, 256, 0, st>>>(a);
    k_lora_expand<T><<<dim3(a.n_rows, (a.n_out + 255) / 256), 256, 0, st>>>(a);
    count_launches(2);
    return cudaGetLastError();
}

}  // namespace
}  // namespace loom

using namespace loom;

extern "C" {

size_t loom_cuda_lora_workspace(const loom_lora_desc *d) { return check(d) ? 0 : ws_bytes_of(d); }

int loom_cuda_lora(const loom_lora_desc *d, const float *d_x, const void *d_a, const void *d_b, const int32_t *d_ranks,
                   const float *d_scales, const int32_t *d_ids, const float *d_base, float *d_out, void *d_ws,
                   size_t ws_bytes, void *stream) {
    if (int rc = rt_need_init()) return rc;
    if (const char *why = check(d)) return rt_decline(why);
    if (d->n_rows == 0) return LOOM_CUDA_OK;
    if (!d_x || !d_out || !d_ids) return rt_decline("lora: x, out and ids are required");
    if (d->n_adapters && d->max_rank && (!d_a || !d_b || !d_ranks || !d_scales))
        return rt_decline("lora: adapters need a, b, ranks and scales");
    if (ws_bytes < ws_bytes_of(d) || (!d_ws && ws_bytes_of(d))) return rt_decline("lora: workspace too small");
    if (reinterpret_cast<uintptr_t>(d_ws) % 16) return rt_decline("lora: workspace not aligned to 16 bytes");
    LoraArgs a{};
    a.x = d_x;
    a.scales = d_scales;
    a.base = d_base;
    a.a = d_a;
    a.b = d_b;
    a.ranks = d_ranks;
    a.ids = d_ids;
    a.out = d_out;
    a.t = static_cast<float *>(d_ws);
    a.x_stride = (int64_t)d->x_stride;
    a.base_stride = (int64_t)d->base_stride;
    a.out_stride = (int64_t)d->out_stride;
    a.a_row = (int64_t)d->a_row_stride;
    a.a_adapter = (int64_t)d->a_adapter_stride;
    a.b_row = (int64_t)d->b_row_stride;
    a.b_adapter = (int64_t)d->b_adapter_stride;
    a.n_rows = (int)d->n_rows;
    a.n_in = (int)d->n_in;
    a.n_out = (int)d->n_out;
    a.n_adapters = (int)(d->max_rank ? d->n_adapters : 0);
    a.max_rank = (int)d->max_rank;
    const cudaError_t e = by_type(d->type, [&](auto t) { return launch<decltype(t)>(a, rt_stream(stream)); });
    return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("lora", e);
}

}  // extern "C"
