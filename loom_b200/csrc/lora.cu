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
// reading the weights. The order of the summed dimension is free, so lane t of a
// row takes its elements 8t .. 8t + 7 of 32, the four products of which use two
// each: operands are read from shared memory 16 bytes at a time.
//
// The two terms of an infinite operand, or of one that rounds to infinity, are an
// infinity and a NaN: every sum that such an operand is part of comes out NaN. A CTA of
// the second kernel that finds a NaN takes its rows again in plain f32, t as well as
// out, which gives the infinity, the large number or the NaN that it stands for.
#include <algorithm>
#include <type_traits>

#include "../../include/loom_cuda.h"
#include "mma.cuh"
#include "serve.cuh"

namespace loom {
namespace {

constexpr int L_RB = 64;   // rows of a block
constexpr int L_NB = 8;    // column tiles (of 8) of a warp's step
constexpr int L_OUT = 128; // output columns of a CTA

struct LoraArgs {
    const float *x, *scales, *base;
    const void *a, *b;
    const int32_t *ranks, *ids;
    float *out, *t;  // t: parts [slice][row][t_row]
    int64_t x_stride, base_stride, out_stride, a_row, a_adapter, b_row, b_adapter;
    int n_rows, n_in, n_out, n_adapters, max_rank, t_row;  // t_row: max_rank, up to a multiple of 4
    int slice, n_slices;
    int wide_x, wide_a, wide_b, wide_out;  // 16-byte (out: 8-byte) accesses are aligned
};

__device__ __forceinline__ int lora_rank(const LoraArgs &a, int id) {
    return id < 0 ? 0 : min(max(a.ranks[id], 0), a.max_rank);
}

// The rows of the j-th adapter (in order of appearance) among a block's rows: their
// count (0: there are fewer adapters), the adapter (-1: none) and the rows in
// s_rows[]. Every warp looks for itself, two rows to a lane, without a barrier;
// the rows are the same in all, and s_rows may be read after the next one.
struct Group {
    int rows, id;
};
__device__ __forceinline__ Group group_of(const LoraArgs &a, int r0, int j, int *s_rows) {
    const int lane = threadIdx.x & 31;
    auto id_of = [&](int r) {
        if (r >= a.n_rows) return -2;
        const int id = a.ids[r];
        return id < 0 || id >= a.n_adapters ? -1 : id;
    };
    const int ia = id_of(r0 + lane), ib = id_of(r0 + 32 + lane);
    const uint32_t ma = __match_any_sync(0xffffffffu, ia), mb = __match_any_sync(0xffffffffu, ib);
    bool second = ib != -2;  // b's first row of its adapter, none among a's
#pragma unroll
    for (int i = 0; i < 32; i++) {
        const int other = __shfl_sync(0xffffffffu, ia, i);  // by all lanes, whatever they have found
        second = second && other != ib;
    }
    const uint32_t below = (1u << lane) - 1;
    const uint32_t fa = __ballot_sync(0xffffffffu, ia != -2 && !(ma & below));
    const uint32_t fb = __ballot_sync(0xffffffffu, second && !(mb & below));
    const int na = __popc(fa);
    if (j >= na + __popc(fb)) return {0, 0};
    // the lane whose row is the j-th first one
    const uint32_t here = __ballot_sync(0xffffffffu, j < na ? ((fa >> lane) & 1) && __popc(fa & below) == j
                                                              : ((fb >> lane) & 1) && __popc(fb & below) == j - na);
    const int id = __shfl_sync(0xffffffffu, j < na ? ia : ib, __ffs(here) - 1);
    const uint32_t ra = __ballot_sync(0xffffffffu, ia == id), rb = __ballot_sync(0xffffffffu, ib == id);
    if (threadIdx.x < 32) {
        if (ia == id) s_rows[__popc(ra & below)] = r0 + lane;
        if (ib == id) s_rows[__popc(ra) + __popc(rb & below)] = r0 + 32 + lane;
    }
    return {__popc(ra) + __popc(rb), id};
}

// A tile of `rows` x `cols` elements (cols a power of two) in shared memory, rows
// `stride` bytes apart, from rows at row_of(j) (null: zeros) of which `n` columns
// exist; 16 bytes at a time, asynchronously where `wide` says that rows lie on 16 bytes
// (`any`: an address there). row_of is asked for a thread's rows in their order.
template <class E, class F>
__device__ __forceinline__ void load_tile(uint8_t *dst, int stride, int rows, int cols, int n, bool wide, F row_of, const E *any) {
    constexpr int N = 16 / (int)sizeof(E);
    const int shift = 31 - __clz(cols / N), c = (threadIdx.x & ((1 << shift) - 1)) * N;  // a thread keeps its columns:
    uint8_t *d = dst + c * (int)sizeof(E);                                               // there are at most 128 pieces a row
    const bool fast = wide && (c + N <= n || c >= n);
    for (int j = threadIdx.x >> shift; j < rows; j += 128 >> shift) {
        const E *src = row_of(j);
        if (fast) {
            const bool in = src && c < n;
            cp_async16(smem_u32(d + j * stride), in ? src + c : any, in);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) reinterpret_cast<E *>(d + j * stride)[k] = src && c + k < n ? src[c + k] : from_f32<E>(0.0f);
        }
    }
}

// eight elements of a tile's row as f32
__device__ __forceinline__ void read8(float (&v)[8], const float *p) {
    const float4 u = *reinterpret_cast<const float4 *>(p), w = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w, v[4] = w.x, v[5] = w.y, v[6] = w.z, v[7] = w.w;
}
// bytes between rows of a tile of `cols` weights: the quarter warps that read 8 rows'
// worth of 16 bytes at once touch every bank
template <class T> __host__ __device__ constexpr int w_stride(int cols) {
    return sizeof(T) == 4 ? cols * 4 + 16 : cols * 2 + (cols == 32 ? 0 : 64);
}

// c[n] += (16 rows x 32) . (32 x 8) for NT column tiles, the lane's eight elements of
// each: rows g and g + 8 split in ah, al, weights of column g of tile n at w + n * 8
// rows of `stride` bytes. The 32 are summed from zero by the tensor core and added to
// c by f32 additions, which round where it truncates; the tiles take turns, since a
// product that adds to the one before it waits for it.
template <class T, int NT>
__device__ __forceinline__ void mma_tiles(float (*c)[4], const uint32_t (&ah)[4][4], const uint32_t (&al)[4][4], const uint8_t *w,
                                          int stride) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1;
    uint4 raw[NT][P];
    float e[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
        for (int p = 0; p < P; p++) raw[n][p] = *reinterpret_cast<const uint4 *>(w + n * 8 * stride + p * 16);
        e[n][0] = e[n][1] = e[n][2] = e[n][3] = 0.0f;
    }
#pragma unroll
    for (int s = 0; s < 4; s++) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 &r = raw[n][s / 2];
                uint32_t bh[2], bl[2];
                split_tf32(__uint_as_float(s % 2 ? r.z : r.x), bh[0], bl[0]);
                split_tf32(__uint_as_float(s % 2 ? r.w : r.y), bh[1], bl[1]);
                mma_tf32(e[n], al[s], bh[0], bh[1]);
                mma_tf32(e[n], ah[s], bl[0], bl[1]);
                mma_tf32(e[n], ah[s], bh[0], bh[1]);
            }
        } else {  // 8 or 11 significant bits: whole in tf32
            uint32_t b[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 &r = raw[n][0];
                const float2 f = unpack2<T>(s == 0 ? r.x : s == 1 ? r.y : s == 2 ? r.z : r.w);
                b[n][0] = __float_as_uint(f.x);
                b[n][1] = __float_as_uint(f.y);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) mma_tf32(e[n], al[s], b[n][0], b[n][1]);
#pragma unroll
            for (int n = 0; n < NT; n++) mma_tf32(e[n], ah[s], b[n][0], b[n][1]);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) c[n][j] += e[n][j];
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
// 16 rows; warps left over split the depth of a tile and join in shared memory. x
// and the weights come in tiles of 32 deep for each of the nk warps that split it,
// through stages of asynchronous copies. A decode batch is bound by latency (32 rows of
// 32 adapters of rank 64, 2,048 wide: 12 us cold), a prompt by issue and latency: 2,048
// f16 rows, 4,096 wide, rank 64 in 38 to 41 us (about 55 TFLOP/s of tf32 products, issue 42 %). 256 threads
// to a CTA (75 against 69 us of the call) and tiles twice as deep (80) were slower.
// bytes of a stage: 64 / nk rows of x and 64 of weights, 32 nk deep; as many stages,
// up to four, as fit what three CTAs of an SM (f32 weights: two) can have
template <class T> __host__ __device__ constexpr int l_xtile(int nk) { return 64 / nk * (128 * nk + 16); }
template <class T> __host__ __device__ constexpr int l_stage(int nk) { return l_xtile<T>(nk) + 64 * w_stride<T>(32 * nk); }
template <class T> __host__ __device__ constexpr int l_smem() { return 2 * l_stage<T>(4); }

template <class T> __global__ void __launch_bounds__(128) k_lora_shrink(LoraArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_rows[L_RB];
    pdl_trigger_();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int i0 = blockIdx.z * a.slice, i1 = min(i0 + a.slice, a.n_in);
    float *part = a.t + (size_t)blockIdx.z * a.n_rows * a.t_row;
    for (int j = blockIdx.y;; j += gridDim.y) {
        __syncthreads();  // the rows of the group before have been read
        const Group gr = group_of(a, blockIdx.x * L_RB, j, s_rows);
        if (!gr.rows) return;
        const int rank = lora_rank(a, gr.id);
        if (!rank) continue;
        __syncthreads();
        const int nk = gr.rows <= 16 ? 4 : gr.rows <= 32 ? 2 : 1, mt = warp / nk, kp = warp % nk, deep = 32 * nk;
        const int xst = deep * 4 + 16, wst = w_stride<T>(deep), tiles = (i1 - i0 + deep - 1) / deep;
        const int size = l_stage<T>(nk), stages = min(l_smem<T>() / size, 4), padded = (gr.rows + 15) / 16 * 16;
        const T *w = static_cast<const T *>(a.a) + gr.id * a.a_adapter;
        const bool busy = mt * 16 < gr.rows;
        // the rows of x that this thread copies: the same in every tile
        const int per = 8 * nk, first = tid / per, every = 128 / per;
        const float *xr[4];
#pragma unroll
        for (int q = 0; q < 4; q++) xr[q] = first + q * every < gr.rows ? a.x + s_rows[first + q * every] * a.x_stride : nullptr;
        for (int k0 = 0; k0 < rank; k0 += L_NB * 8) {
            const int cols = min(rank - k0, L_NB * 8);
            auto fetch = [&](int i) {
                if (i < tiles) {
                    uint8_t *st = smem + i % stages * size;
                    const int at = i0 + i * deep;
                    int q = 0;
                    load_tile<float>(st, xst, padded, deep, i1 - at, a.wide_x, [&](int r) {
                        const float *x = q == 0 ? xr[0] : q == 1 ? xr[1] : q == 2 ? xr[2] : xr[3];
                        q++;
                        return r < gr.rows ? x + at : (const float *)nullptr;
                    }, a.x);
                    load_tile<T>(st + l_xtile<T>(nk), wst, cols > 32 ? 64 : (cols + 15) / 16 * 16, deep, i1 - at, a.wide_a,
                                 [&](int r) { return r < cols ? w + (k0 + r) * a.a_row + at : (const T *)nullptr; }, w);
                }
                cp_async_commit();
            };
            float c[L_NB][4];
#pragma unroll
            for (int n = 0; n < L_NB; n++) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.0f;
            __syncthreads();  // the sums of the ranks before have been read
            for (int i = 0; i < stages - 1; i++) fetch(i);
            for (int i = 0; i < tiles; i++) {
                if (stages == 4) cp_async_wait<2>();
                else if (stages == 3) cp_async_wait<1>();
                else cp_async_wait<0>();
                __syncthreads();
                fetch(i + stages - 1);  // into the stage that was read in the step before
                const uint8_t *st = smem + i % stages * size;
                if (busy) {
                    float ua[8], ub[8];
                    uint32_t ah[4][4], al[4][4];
                    const float *x = reinterpret_cast<const float *>(st + (mt * 16 + g) * xst) + kp * 32 + 8 * t;
                    read8(ua, x);
                    read8(ub, x + 8 * (xst / 4));
                    split_rows(ah, al, ua, ub);
                    const uint8_t *ws = st + l_xtile<T>(nk) + g * wst + (kp * 32 + 8 * t) * (int)sizeof(T);
                    if (cols > 32) {
                        mma_tiles<T, 4>(c, ah, al, ws, wst);
                        mma_tiles<T, 4>(c + 4, ah, al, ws + 32 * wst, wst);
                    } else if (cols > 16) {
                        mma_tiles<T, 4>(c, ah, al, ws, wst);
                    } else {
                        mma_tiles<T, 2>(c, ah, al, ws, wst);
                    }
                }
            }
            cp_async_wait<0>();
            if (nk == 1) {  // a warp has its rows' whole sums
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int m = mt * 16 + g + 8 * h;
                    if (m >= gr.rows) continue;
                    float *p = part + (size_t)s_rows[m] * a.t_row + k0 + 2 * t;
#pragma unroll
                    for (int n = 0; n < L_NB; n++) {
                        if (n * 8 + 2 * t < cols) p[n * 8] = c[n][2 * h];
                        if (n * 8 + 2 * t + 1 < cols) p[n * 8 + 1] = c[n][2 * h + 1];
                    }
                }
                continue;
            }
            __syncthreads();
            float(*s_t)[16][L_NB * 8 + 1] = reinterpret_cast<float(*)[16][L_NB * 8 + 1]>(smem);
#pragma unroll
            for (int n = 0; n < L_NB; n++) {
                s_t[warp][g][n * 8 + 2 * t] = c[n][0];
                s_t[warp][g][n * 8 + 2 * t + 1] = c[n][1];
                s_t[warp][g + 8][n * 8 + 2 * t] = c[n][2];
                s_t[warp][g + 8][n * 8 + 2 * t + 1] = c[n][3];
            }
            __syncthreads();
            for (int m = warp; m < gr.rows; m += 4)
                for (int k = lane; k < cols; k += 32) {
                    float s = 0.0f;
                    for (int q = 0; q < nk; q++) s += s_t[(m / 16) * nk + q][m % 16][k];
                    part[(size_t)s_rows[m] * a.t_row + k0 + k] = s;
                }
        }
    }
}

// out: CTA (block of rows, adapter of the block, L_OUT columns). A warp has 16 rows;
// warps left over split the columns. The weights and the base, which do not wait for
// t, are asked for before it. Bound by latency: 2,048 rows and columns of rank 64 in 33
// us (1 TB/s of base and out); several column chunks to a CTA took 72 us of a call,
// not 69.
constexpr int L_DEEP = 64;  // ranks at a time
template <class T> constexpr size_t l_expand_smem() { return (size_t)L_OUT * w_stride<T>(L_DEEP) + 64 * (L_DEEP * 4 + 16); }

// A CTA's rows and columns in plain f32 (s_x: room for L_DEEP of t). A call of its own:
// inlined, it cost 2,048 rows 2 us. A NaN in one of 2,048 rows makes the call take 1.1
// ms, in all of them 9 ms.
template <class T> __device__ __noinline__ void expand_plain(const LoraArgs &a, Group gr, const int *s_rows, float *s_x, int o0) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = lora_rank(a, gr.id), o = o0 + tid;
    const bool in = o < a.n_out;
    const float scale = a.scales[gr.id];
    const T *wa = static_cast<const T *>(a.a) + gr.id * a.a_adapter, *wb = static_cast<const T *>(a.b) + gr.id * a.b_adapter + o * a.b_row;
    for (int m = 0; m < gr.rows; m++) {
        const int64_t row = s_rows[m];
        const float *x = a.x + row * a.x_stride, *t = a.t + row * a.t_row;
        float s = in && a.base ? a.base[row * a.base_stride + o] : 0.0f;
        for (int k0 = 0; k0 < rank; k0 += L_DEEP) {
            const int n = min(rank - k0, L_DEEP);
            __syncthreads();
            if (tid < n) {
                float v = 0.0f;
#pragma unroll 4
                for (int z = 0; z < a.n_slices; z++) v += __ldcg(t + (size_t)z * a.n_rows * a.t_row + k0 + tid);
                s_x[tid] = v;
            }
            __syncthreads();
            for (int k = warp; k < n; k += 4) {
                if (s_x[k] == s_x[k]) continue;
                const T *w = wa + (k0 + k) * a.a_row;
                float v = 0.0f;
#pragma unroll 4
                for (int i = lane; i < a.n_in; i += 32) v = fmaf(x[i], to_f32(w[i]), v);
                v = warp_sum(v);
                __syncwarp();
                if (lane == 0) s_x[k] = v;
            }
            __syncthreads();
#pragma unroll 4
            for (int k = 0; k < n && in; k++) s = fmaf(to_f32(wb[k0 + k]), s_x[k] * scale, s);
        }
        if (in) a.out[row * a.out_stride + o] = s;
    }
}

template <class T> __global__ void __launch_bounds__(128) k_lora_expand(const __grid_constant__ LoraArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ int s_rows[L_RB];
    constexpr int WST = w_stride<T>(L_DEEP), TST = L_DEEP + 4;
    float *s_x = reinterpret_cast<float *>(smem + L_OUT * WST);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    for (int grp = blockIdx.y;; grp += gridDim.y) {
        __syncthreads();  // the rows and tiles of the group before have been read
        const Group gr = group_of(a, blockIdx.x * L_RB, grp, s_rows);
        if (!gr.rows) break;
        __syncthreads();
        const int rank = lora_rank(a, gr.id);
        const float scale = rank ? a.scales[gr.id] : 0.0f;
        const int o0 = blockIdx.z * L_OUT, outs = min(L_OUT, a.n_out - o0);
        const T *w = static_cast<const T *>(a.b) + (rank ? gr.id : 0) * a.b_adapter + o0 * a.b_row;
        auto weights = [&](int k) {
            const int deep = min((rank - k + 31) / 32 * 32, L_DEEP);
            load_tile<T>(smem, WST, L_OUT, deep, rank - k, a.wide_b,
                         [&](int j) { return j < outs ? w + j * a.b_row + k : (const T *)nullptr; }, w);
            cp_async_commit();
        };
        if (rank) weights(0);
        const int nc = gr.rows <= 16 ? 4 : gr.rows <= 32 ? 2 : 1, mt = warp / nc, cp = warp % nc;
        const bool in[2] = {mt * 16 + g < gr.rows, mt * 16 + g + 8 < gr.rows};
        const int64_t row[2] = {in[0] ? s_rows[mt * 16 + g] : 0, in[1] ? s_rows[mt * 16 + g + 8] : 0};
        auto go = [&](auto tiles) {
            constexpr int NT = decltype(tiles)::value;  // column tiles of 8
            const int c0 = cp * NT * 8;
            float c[NT][4];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int o = c0 + n * 8 + 2 * t;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float2 b = make_float2(0.0f, 0.0f);
                    if (in[h] && a.base) {
                        const float *p = a.base + row[h] * a.base_stride + o0 + o;
                        if (a.wide_out && o + 1 < outs) {
                            b = *reinterpret_cast<const float2 *>(p);
                        } else {
                            if (o < outs) b.x = p[0];
                            if (o + 1 < outs) b.y = p[1];
                        }
                    }
                    c[n][2 * h] = b.x;
                    c[n][2 * h + 1] = b.y;
                }
            }
            auto clear = [&](int deep, int d4) {  // what the tile has beside the sums
                for (int j = tid; j < (gr.rows + 15) / 16 * 16 * (deep / 4); j += 128) {
                    const int m = j / (deep / 4), q = j % (deep / 4);
                    if (m >= gr.rows || q >= d4) *reinterpret_cast<float4 *>(s_x + m * TST + q * 4) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            };
            if (rank) clear(min((rank + 31) / 32 * 32, L_DEEP), (min(rank, L_DEEP) + 3) / 4);
            pdl_wait_();  // t is there
            for (int k = 0; k < rank; k += L_DEEP) {
                const int deep = min((rank - k + 31) / 32 * 32, L_DEEP);
                if (k) {
                    __syncthreads();
                    weights(k);
                }
                // the parts' sums, four ranks of a row to a thread
                const size_t next = (size_t)a.n_rows * a.t_row;  // from part to part
                const int d4 = (min(rank - k, deep) + 3) / 4;
                if (k) clear(deep, d4);
                for (int j = tid; j < gr.rows * d4; j += 128) {
                    const int m = j / d4, q = j % d4 * 4, left = rank - k - q;  // what lies past the rank was not written
                    const float *p = a.t + (size_t)s_rows[m] * a.t_row + k + q;
                    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int z = 0; z < a.n_slices; z++) {
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + z * next));
                        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
                    }
                    *reinterpret_cast<float4 *>(s_x + m * TST + q) = make_float4(
                        s.x * scale, left > 1 ? s.y * scale : 0.0f, left > 2 ? s.z * scale : 0.0f, left > 3 ? s.w * scale : 0.0f);
                }
                cp_async_wait<0>();
                __syncthreads();
                if (mt * 16 < gr.rows)
                    for (int q = 0; q < deep; q += 32) {
                        float ua[8], ub[8];
                        uint32_t ah[4][4], al[4][4];
                        read8(ua, s_x + (mt * 16 + g) * TST + q + 8 * t);
                        read8(ub, s_x + (mt * 16 + g + 8) * TST + q + 8 * t);
                        split_rows(ah, al, ua, ub);
#pragma unroll
                        for (int n = 0; n < NT; n += 4)
                            mma_tiles<T, 4>(c + n, ah, al, smem + (c0 + n * 8 + g) * WST + (q + 8 * t) * (int)sizeof(T), WST);
                    }
            }
            bool nan = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) nan = nan || c[n][j] != c[n][j];
            if (__syncthreads_or(nan && rank)) {  // none has written yet: out may be base
                expand_plain<T>(a, gr, s_rows, s_x, o0);
                return;
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int o = c0 + n * 8 + 2 * t;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (!in[h]) continue;
                    float *p = a.out + row[h] * a.out_stride + o0 + o;
                    if (a.wide_out && o + 1 < outs) {
                        *reinterpret_cast<float2 *>(p) = make_float2(c[n][2 * h], c[n][2 * h + 1]);
                    } else {
                        if (o < outs) p[0] = c[n][2 * h];
                        if (o + 1 < outs) p[1] = c[n][2 * h + 1];
                    }
                }
            }
        };
        if (nc == 4) go(std::integral_constant<int, L_OUT / 32>{});
        else if (nc == 2) go(std::integral_constant<int, L_OUT / 16>{});
        else go(std::integral_constant<int, L_OUT / 8>{});
    }
    pdl_wait_();  // also where there was nothing to do
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
// are prompts, whose rows come in runs of one. Two CTAs per SM: at one and at four a
// prompt of 2,048 rows took 86 and 66 us, here 62, 32 decode rows 21.3 and 17.0, here
// 17.5. Slices of 128 at the least: of 256, 168 rows of 4,096 took 20.6 us, not 18.6;
// of 64 19.4, not 17.0.
int slice_of(const loom_lora_desc *d) {
    const size_t blocks = (d->n_rows + L_RB - 1) / L_RB;
    const size_t groups = blocks > 1 ? blocks : std::max<size_t>(1, std::min(d->n_rows, d->n_adapters));
    const size_t want = std::max<size_t>(1, (2 * 148 + groups - 1) / groups);
    return (int)std::max<size_t>(128, ((d->n_in + want - 1) / want + 127) / 128 * 128);
}
size_t slices_of(const loom_lora_desc *d) { return (d->n_in + slice_of(d) - 1) / slice_of(d); }
size_t t_row_of(const loom_lora_desc *d) { return (d->max_rank + 3) / 4 * 4; }
size_t ws_bytes_of(const loom_lora_desc *d) { return slices_of(d) * d->n_rows * t_row_of(d) * sizeof(float); }

template <class T> cudaError_t launch(const LoraArgs &a, cudaStream_t st) {
    const unsigned blocks = (a.n_rows + L_RB - 1) / L_RB, most = std::min(std::min(L_RB, a.n_rows), a.n_adapters + 1);
    // A CTA per adapter of a decode batch's one block; of a prompt's blocks, whose rows
    // come in runs, as many as fill the GPU, each taking several adapters in turn where
    // there are more (at 2, 4, 6 and 12 CTAs per SM 2,048 rows took 67, 67, 62 and 64 us).
    auto groups = [&](unsigned others) { return blocks == 1 ? most : std::min(most, std::max(2u, 6 * 148 / (blocks * others))); };
    cudaError_t e = allow_smem<k_lora_expand<T>>(l_expand_smem<T>());
    if (e != cudaSuccess) return e;
    if (a.n_adapters) {
        constexpr size_t smem = l_smem<T>();
        if ((e = allow_smem<k_lora_shrink<T>>(smem)) != cudaSuccess) return e;
        k_lora_shrink<T><<<dim3(blocks, groups(a.n_slices), a.n_slices), 128, smem, st>>>(a);
        count_launch();
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    const unsigned outs = (a.n_out + L_OUT - 1) / L_OUT;
    const dim3 grid(blocks, groups(outs), outs);
    if (a.n_adapters) return launch_pdl_(k_lora_expand<T>, grid, dim3(128), l_expand_smem<T>(), st, a);
    k_lora_expand<T><<<grid, 128, l_expand_smem<T>(), st>>>(a);  // reads ids before its wait: only behind this call's own kernel
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
    a.t_row = (int)t_row_of(d);
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
