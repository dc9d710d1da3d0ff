// lora.cu -- low-rank adapters of many requests at once
// (include/loom_cuda.h, loom_cuda_lora):
//
//   out[r] = base[r] + scale_a * B_a (A_a x[r]),  a = ids[r]
//
// Two kernels: t[r] = A_a x[r] (the width n_in in slices, a part per slice), then
// out[r] = base[r] + B_a (scale_a * sum of the parts). A CTA takes the rows of one
// adapter within a block of 64 rows, found from the ids by the CTA itself, so an
// adapter's weights are read once per block whatever its rows' order: a decode
// batch is one block, a prompt's rows come in runs. A row with no adapter keeps
// its base.
//
// Both products run on the tensor cores with 16 rows to a fragment, x, t and f32
// weights as two tf32 terms (mma.cuh; 16-bit weights are exact in one), since
// they would otherwise be bound by their multiply-adds as soon as some rows share
// an adapter; few rows leave most of a fragment idle, but those are bound by
// reading the weights. Operands come straight from global memory in 16-byte
// pieces: the order of the summed dimension is free, so lane t of a row takes
// its elements 8t .. 8t + 7 of 32, the four products of which use two each.
#include <algorithm>

#include "../../include/loom_cuda.h"
#include "mma.cuh"
#include "serve.cuh"

namespace loom {
namespace {

constexpr int L_RB = 64;   // rows of a block
constexpr int L_NB = 8;    // column tiles (of 8) of a warp's step
constexpr int L_OUT = 256; // output columns of a CTA

struct LoraArgs {
    const float *x, *scales, *base;
    const void *a, *b;
    const int32_t *ranks, *ids;
    float *out, *t;  // t: parts [slice][row][max_rank]
    int64_t x_stride, base_stride, out_stride, a_row, a_adapter, b_row, b_adapter;
    int n_rows, n_in, n_out, n_adapters, max_rank;
    int slice, n_slices;
    int wide_x, wide_a, wide_b, wide_out;  // 16-byte (out: 8-byte) accesses are aligned
};

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int id) {
    return id < 0 ? 0 : min(max(a.ranks[id], 0), a.max_rank);
}

// The rows of the j-th adapter (in order of appearance) among the block's rows:
// their count (0: there are fewer adapters), in s_rows[]; id -1 stands for none.
struct Group {
    int rows, id;
};
__device__ __forceinline__ Group group_of(const LoraArgs &a, int r0, int j, int *s_ids, int *s_rows) {
    __shared__ int s_id, s_n;
    __shared__ uint32_t s_mask[2];
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < L_RB) {
        int id = r0 + tid < a.n_rows ? a.ids[r0 + tid] : -2;
        if (id != -2 && (id < 0 || id >= a.n_adapters)) id = -1;
        if (r0 + tid >= a.n_rows) id = -2;
        s_ids[tid] = id;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    bool first = false;
    if (tid < L_RB) {
        first = s_ids[tid] != -2;
        for (int i = 0; i < tid && first; i++) first = s_ids[i] != s_ids[tid];
        const uint32_t m = __ballot_sync(0xffffffffu, first);
        if (lane == 0) s_mask[tid >> 5] = m;
    }
    __syncthreads();
    if (first && (tid < 32 ? 0 : __popc(s_mask[0])) + __popc(s_mask[tid >> 5] & ((1u << lane) - 1)) == j) {
        s_id = s_ids[tid];
        s_n = 1;
    }
    __syncthreads();
    if (!s_n) return {0, 0};
    const int id = s_id;
    bool mine = false;
    if (tid < L_RB) {
        mine = s_ids[tid] == id;
        const uint32_t m = __ballot_sync(0xffffffffu, mine);
        if (lane == 0) s_mask[tid >> 5] = m;
    }
    __syncthreads();
    if (mine) s_rows[(tid < 32 ? 0 : __popc(s_mask[0])) + __popc(s_mask[tid >> 5] & ((1u << lane) - 1))] = r0 + tid;
    const int n = __popc(s_mask[0]) + __popc(s_mask[1]);
    __syncthreads();
    return {n, id};
}

// elements i .. i + 7 of p as f32, zeros from n on; two 16-byte reads (one for
// 16-bit types) where that is aligned
__device__ __forceinline__ void load8(float (&v)[8], const float *p, int i, int n, bool wide) {
    if (wide && i + 8 <= n) {
        const float4 u = __ldg(reinterpret_cast<const float4 *>(p + i)), w = __ldg(reinterpret_cast<const float4 *>(p + i + 4));
        v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w, v[4] = w.x, v[5] = w.y, v[6] = w.z, v[7] = w.w;
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i + k < n ? p[i + k] : 0.0f;
    }
}
template <class T> __device__ __forceinline__ void load8(float (&v)[8], const T *p, int i, int n, bool wide) {
    if (wide && i + 8 <= n) {
        const uint4 u = ld_v4(p + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 f = unpack2<T>(w[k]);
            v[2 * k] = f.x, v[2 * k + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = i + k < n ? to_f32(p[i + k]) : 0.0f;
    }
}

// c += (16 rows x 32) . (32 x 8) for the lane's eight elements of each operand:
// ua, ub of rows g and g + 8, w of column g. The 32 are summed from zero by the
// tensor core and added to c by f32 additions, which round where it truncates.
template <class T>
__device__ __forceinline__ void mma_32(float (&c)[4], const uint32_t (&ah)[4][4], const uint32_t (&al)[4][4], const float (&w)[8]) {
    float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; s++) {
        if constexpr (sizeof(T) == 4) {
            uint32_t bh[2], bl[2];
            split_tf32(w[2 * s], bh[0], bl[0]);
            split_tf32(w[2 * s + 1], bh[1], bl[1]);
            mma_tf32(e, al[s], bh[0], bh[1]);
            mma_tf32(e, ah[s], bl[0], bl[1]);
            mma_tf32(e, ah[s], bh[0], bh[1]);
        } else {  // 8 or 11 significant bits: whole in tf32
            const uint32_t b0 = __float_as_uint(w[2 * s]), b1 = __float_as_uint(w[2 * s + 1]);
            mma_tf32(e, al[s], b0, b1);
            mma_tf32(e, ah[s], b0, b1);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) c[j] += e[j];
}
__device__ __forceinline__ void split_rows(uint32_t (&ah)[4][4], uint32_t (&al)[4][4], const float (&ua)[8], const float (&ub)[8]) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
        split_tf32(ua[2 * s], ah[s][0], al[s][0]);
        split_tf32(ub[2 * s], ah[s][1], al[s][1]);
        split_tf32(ua[2 * s + 1], ah[s][2], al[s][2]);
        split_tf32(ub[2 * s + 1], ah[s][3], al[s][3]);
    }
}

// Parts of t: CTA (block of rows, adapter of the block, slice of n_in). A warp has
// 16 rows; warps left over split the slice and join in shared memory.
template <class T> __global__ void __launch_bounds__(128) k_lora_shrink(LoraArgs a) {
    __shared__ int s_ids[L_RB], s_rows[L_RB];
    __shared__ float s_t[4][16][L_NB * 8 + 1];
    pdl_trigger_();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const Group gr = group_of(a, blockIdx.x * L_RB, blockIdx.y, s_ids, s_rows);
    const int rank = gr.rows ? lora_rank(a, gr.id) : 0;
    if (!rank) return;
    const int nk = gr.rows <= 16 ? 4 : gr.rows <= 32 ? 2 : 1, mt = warp / nk, kp = warp % nk;
    const int i0 = blockIdx.z * a.slice, i1 = min(i0 + a.slice, a.n_in);
    const bool ina = mt * 16 + g < gr.rows, inb = mt * 16 + g + 8 < gr.rows;
    const float *xa = a.x + (ina ? s_rows[mt * 16 + g] : 0) * a.x_stride;
    const float *xb = a.x + (inb ? s_rows[mt * 16 + g + 8] : 0) * a.x_stride;
    const T *w = static_cast<const T *>(a.a) + gr.id * a.a_adapter;
    float *part = a.t + (size_t)blockIdx.z * a.n_rows * a.max_rank;
    for (int k0 = 0; k0 < rank; k0 += L_NB * 8) {
        float c[L_NB][4];
#pragma unroll
        for (int n = 0; n < L_NB; n++) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
        if (mt * 16 < gr.rows) {
            for (int i = i0 + kp * 32; i < i1; i += nk * 32) {
                float ua[8], ub[8];
                load8(ua, xa, i + 8 * t, ina ? i1 : 0, a.wide_x);
                load8(ub, xb, i + 8 * t, inb ? i1 : 0, a.wide_x);
                float v[L_NB][8];
#pragma unroll
                for (int n = 0; n < L_NB; n++)
                    load8(v[n], w + (k0 + n * 8 + g) * a.a_row, i + 8 * t, k0 + n * 8 + g < rank ? i1 : 0, a.wide_a);
                uint32_t ah[4][4], al[4][4];
                split_rows(ah, al, ua, ub);
#pragma unroll
                for (int n = 0; n < L_NB; n++)
                    if (k0 + n * 8 < rank) mma_32<T>(c[n], ah, al, v[n]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < L_NB; n++) {
            s_t[warp][g][n * 8 + 2 * t] = c[n][0];
            s_t[warp][g][n * 8 + 2 * t + 1] = c[n][1];
            s_t[warp][g + 8][n * 8 + 2 * t] = c[n][2];
            s_t[warp][g + 8][n * 8 + 2 * t + 1] = c[n][3];
        }
        __syncthreads();
        const int cols = min(rank - k0, L_NB * 8);
        for (int j = tid; j < gr.rows * cols; j += 128) {
            const int m = j / cols, k = j % cols;
            float s = 0.0f;
            for (int q = 0; q < nk; q++) s += s_t[(m / 16) * nk + q][m % 16][k];
            part[(size_t)s_rows[m] * a.max_rank + k0 + k] = s;
        }
    }
}

// out: CTA (block of rows, adapter of the block, L_OUT columns); a warp has a
// quarter of the columns, for all the rows.
template <class T> __global__ void __launch_bounds__(128) k_lora_expand(LoraArgs a) {
    extern __shared__ float s_x[];  // t of the group's rows [64][stride]
    __shared__ int s_ids[L_RB], s_rows[L_RB];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const Group gr = group_of(a, blockIdx.x * L_RB, blockIdx.y, s_ids, s_rows);
    pdl_wait_();
    if (!gr.rows) return;
    const int rank = lora_rank(a, gr.id), deep = (rank + 31) / 32 * 32, stride = a.max_rank + 36;
    const float scale = rank ? a.scales[gr.id] : 0.0f;
    for (int j = tid; j < (gr.rows + 15) / 16 * 16 * deep; j += 128) {
        const int m = j / deep, k = j % deep;
        float s = 0.0f;
        if (m < gr.rows && k < rank)
            for (int z = 0; z < a.n_slices; z++) s += a.t[((size_t)z * a.n_rows + s_rows[m]) * a.max_rank + k];
        s_x[m * stride + k] = s * scale;
    }
    __syncthreads();
    const int o0 = blockIdx.z * L_OUT + warp * (L_OUT / 4);
    const T *w = static_cast<const T *>(a.b) + (rank ? gr.id : 0) * a.b_adapter;
    for (int m0 = 0; m0 < gr.rows; m0 += 16) {
        float c[L_NB][4];
        const bool in[2] = {m0 + g < gr.rows, m0 + g + 8 < gr.rows};
        const int64_t row[2] = {in[0] ? s_rows[m0 + g] : 0, in[1] ? s_rows[m0 + g + 8] : 0};
#pragma unroll
        for (int n = 0; n < L_NB; n++) {
            const int o = o0 + n * 8 + 2 * t;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                float2 b = make_float2(0.0f, 0.0f);
                if (in[h] && a.base) {
                    const float *p = a.base + row[h] * a.base_stride + o;
                    if (a.wide_out && o + 1 < a.n_out)
                        b = *reinterpret_cast<const float2 *>(p);
                    else {
                        if (o < a.n_out) b.x = p[0];
                        if (o + 1 < a.n_out) b.y = p[1];
                    }
                }
                c[n][2 * h] = b.x;
                c[n][2 * h + 1] = b.y;
            }
        }
        for (int k = 0; k < rank; k += 32) {
            uint32_t ah[4][4], al[4][4];
            float ua[8], ub[8];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                ua[q] = s_x[(m0 + g) * stride + k + 8 * t + q];
                ub[q] = s_x[(m0 + g + 8) * stride + k + 8 * t + q];
            }
            split_rows(ah, al, ua, ub);
            float v[L_NB][8];
#pragma unroll
            for (int n = 0; n < L_NB; n++)
                load8(v[n], w + (int64_t)(o0 + n * 8 + g) * a.b_row, k + 8 * t, o0 + n * 8 + g < a.n_out ? rank : 0, a.wide_b);
#pragma unroll
            for (int n = 0; n < L_NB; n++) mma_32<T>(c[n], ah, al, v[n]);
        }
#pragma unroll
        for (int n = 0; n < L_NB; n++) {
            const int o = o0 + n * 8 + 2 * t;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (!in[h]) continue;
                float *p = a.out + row[h] * a.out_stride + o;
                if (a.wide_out && o + 1 < a.n_out)
                    *reinterpret_cast<float2 *>(p) = make_float2(c[n][2 * h], c[n][2 * h + 1]);
                else {
                    if (o < a.n_out) p[0] = c[n][2 * h];
                    if (o + 1 < a.n_out) p[1] = c[n][2 * h + 1];
                }
            }
        }
    }
}

const char *check(const loom_lora_desc *d) {
    if (!d) return "lora: no descriptor";
    if (!elem_bytes(d->type)) return "lora: type must be LOOM_F32, LOOM_F16 or LOOM_BF16";
    if (!d->n_in || !d->n_out || d->n_in > (1u << 22) || d->n_out > (1u << 22)) return "lora: widths must be 1..2^22";
    if (d->n_rows > (1u << 24)) return "lora: at most 2^24 rows";
    if (d->n_adapters > (1u << 20)) return "lora: at most 2^20 adapters";
    if (d->max_rank > 512) return "lora: max_rank must be at most 512";
    return nullptr;
}

// Slices of n_in: enough CTAs for the GPU's 148 SMs, at least 128 wide. One block
// is a decode batch, where about every row brings its own adapter; more blocks
// are prompts, whose rows come in runs of one.
int slice_of(const loom_lora_desc *d) {
    const size_t blocks = (d->n_rows + L_RB - 1) / L_RB;
    const size_t groups = blocks > 1 ? blocks : std::max<size_t>(1, std::min(d->n_rows, d->n_adapters));
    const size_t want = std::max<size_t>(1, (2 * 148 + groups - 1) / groups);
    return (int)std::max<size_t>(128, ((d->n_in + want - 1) / want + 127) / 128 * 128);
}
size_t slices_of(const loom_lora_desc *d) { return (d->n_in + slice_of(d) - 1) / slice_of(d); }
size_t ws_bytes_of(const loom_lora_desc *d) { return slices_of(d) * d->n_rows * d->max_rank * sizeof(float); }

template <class T> cudaError_t launch(const LoraArgs &a, cudaStream_t st) {
    const unsigned blocks = (a.n_rows + L_RB - 1) / L_RB, groups = std::min(std::min(L_RB, a.n_rows), a.n_adapters + 1);
    if (a.n_adapters) {
        k_lora_shrink<T><<<dim3(blocks, groups, a.n_slices), 128, 0, st>>>(a);
        count_launch();
        if (const cudaError_t e = cudaGetLastError(); e != cudaSuccess) return e;
    }
    const size_t smem = (size_t)L_RB * (a.max_rank + 36) * sizeof(float);
    cudaError_t e = allow_smem<k_lora_expand<T>>(smem);
    if (e != cudaSuccess) return e;
    const dim3 grid(blocks, groups, (a.n_out + L_OUT - 1) / L_OUT);
    if (a.n_adapters) return launch_pdl_(k_lora_expand<T>, grid, dim3(128), smem, st, a);
    k_lora_expand<T><<<grid, 128, smem, st>>>(a);  // reads ids before its wait: only behind this call's own kernel
    count_launch();
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
    a.slice = slice_of(d);
    a.n_slices = (int)slices_of(d);
    const size_t size = elem_bytes(d->type);
    auto aligned = [](const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
    a.wide_x = aligned(d_x, 16) && d->x_stride % 4 == 0;
    a.wide_a = aligned(d_a, 16) && d->a_row_stride * size % 16 == 0 && d->a_adapter_stride * size % 16 == 0;
    a.wide_b = aligned(d_b, 16) && d->b_row_stride * size % 16 == 0 && d->b_adapter_stride * size % 16 == 0;
    a.wide_out = aligned(d_out, 8) && d->out_stride % 2 == 0 && (!d_base || (aligned(d_base, 8) && d->base_stride % 2 == 0));
    const cudaError_t e = by_type(d->type, [&](auto t) { return launch<decltype(t)>(a, rt_stream(stream)); });
    return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("lora", e);
}

}  // extern "C"
