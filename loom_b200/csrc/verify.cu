// verify.cu -- verification of drafted tokens against the target's
// probabilities, from given random numbers (include/loom_cuda.h,
// loom_cuda_verify).
//
// Sequence b has the rows r0 .. r1-1 of logits: its last token's and those of
// its drafts. Draft j (tokens[r0 + j], j = 1 ..) is judged by row r = r0 + j - 1:
//
//   p = softmax(logits[r] / T), q = draft_probs[r]   (q = 1 at the draft without them)
//   accepted while u[r] q(d) < p(d); at temperature 0 while d is the argmax
//
// then one token from the first row that is not followed by an accepted draft:
// after a refusal from max(p - q, 0), after the last draft from p, at the first
// index whose running sum exceeds u[r1 - 1] times the whole sum. Accepting with
// min(1, p / q) and drawing from the rest leaves the target's distribution.
//
// The sums behind that choice are 64 bits wide: neighbours of a 150,000-entry
// vocabulary lie 1e-6 apart in the running sum, where a 32-bit sum's rounding,
// not the random number, would choose.
#include <type_traits>

#include "../../include/loom_cuda.h"
#include "serve.cuh"

namespace loom {
namespace {

constexpr int V_C = 8, V_W = 16, V_T = V_W * 32;  // CTAs of a cluster, warps of a CTA

// One CTA's part of a row; row_stat reads a row's parts as one
struct RowPart {
    double z;   // sum of e^((l - top) / T) over its logits
    float top;  // the row's largest logit, or the part's own (two passes); -inf when none is above it
    int arg;    // first index of the row's largest among its logits (greedy rows), or 2^31 - 1
};
struct RowStat {
    float top, z;
    int arg;
};

struct VerifyArgs {
    const void *logits;
    const float *probs, *u, *temp;
    const int32_t *tokens;
    const uint32_t *seq_rows;
    int32_t *out, *n_out;
    float *logprobs;
    RowPart *stat;  // [rows][parts]
    int64_t logits_stride, probs_stride;
    int n_seqs, n_rows, vocab, parts, two;  // two: the parts are of the two passes
};

__device__ __forceinline__ float temp_of(const VerifyArgs &a, int b) { return a.temp ? a.temp[b] : 1.0f; }
// 1 / T; a greedy sequence's probabilities (its log-probabilities' base) are those of T = 1
__device__ __forceinline__ float inv_temp(float t) { return t <= 0.0f ? 1.0f : __fdiv_rn(1.0f, t); }
// e^((l - top) / T): NaN weighs nothing, as the greedy sampler never takes it
__device__ __forceinline__ float weight(float l, float top, float inv) {
    if (l == top) return top == -INFINITY ? 0.0f : 1.0f;
    const float e = expf(fmul(fsub(l, top), inv));
    return e == e ? e : 0.0f;
}

__device__ __forceinline__ double running(double v) {  // sum over the lanes up to this one
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// the sequence of row r: the last b with seq_rows[b] <= r
__device__ __forceinline__ int seq_of(const VerifyArgs &a, int r) {
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.seq_rows[mid] <= (uint32_t)r) lo = mid; else hi = mid;
    }
    return lo;
}

// of row r, by a whole warp
__device__ __forceinline__ RowStat row_stat(const VerifyArgs &a, int r) {
    const RowPart *p = a.stat + (size_t)r * a.parts;
    double z = 0.0;
    float top = -INFINITY;
    int arg = 0x7FFFFFFF;
    for (int i = threadIdx.x & 31; i < a.parts; i += 32) {
        z += p[i].z;
        top = fmaxf(top, p[i].top);
        arg = min(arg, p[i].arg);
    }
    arg = __reduce_min_sync(0xffffffffu, arg);
    return {warp_max(top), (float)warp_sum_d(z), arg == 0x7FFFFFFF ? 0 : arg};
}

// ---- layout of a row over a cluster -----------------------------------------------
// A row of logits is spread over a cluster of V_C CTAs of V_W warps: warp k of the
// cluster's V_C * V_W has the k-th run of `run` 16-byte pieces, its lane l the
// pieces l, l + 32, ... of the run. So a running sum over the vocabulary is one
// over the warps, then over groups of 32 pieces, then over lanes. A thread keeps
// its first v_nv pieces in registers, so the row crosses the memory once although the
// weights need its maximum; what is left is read again. Rows that take one launch have
// up to 400 KB (two_passes below), 7 pieces a thread: f32 keeps all of them, 16-bit
// types, twice the logits in each, 5. Only calls of more than 65,535 rows, which the
// two passes' grid does not hold, bring longer ones. A row that does not start on 16
// bytes is shifted: its first piece holds fewer logits.
template <class T> constexpr int v_nv() { return sizeof(T) == 4 ? 7 : 5; }

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
// the address in CTA `rank` of a variable of this CTA's shared memory
__device__ __forceinline__ uint32_t peer(const void *p, unsigned rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float peer_ldf(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ double peer_ldd(uint32_t a) {
    double v;
    asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(a) : "memory");
    return v;
}

// two f32 at once (one issue slot, each half rounded as by itself)
struct F2 {
    uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 split(F2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// A sum of weights in [0, 1] as exact as a 64-bit one, without its conversions:
// each is cut at 2^-16; the upper parts, up to 256 of them, add exactly in f32, the
// lower ones, 2^-17 at most, with an error below 2^-31.
struct Sum01 {
    F2 hi = f2(0.0f, 0.0f), lo = f2(0.0f, 0.0f);
    __device__ __forceinline__ void add(F2 e) {
        const F2 up = (e + f2(128.0f, 128.0f)) + f2(-128.0f, -128.0f);
        hi = hi + up;
        lo = lo + (e + up * f2(-1.0f, -1.0f));
    }
    __device__ __forceinline__ double get() const {
        const float2 h = split(hi), l = split(lo);
        return ((double)h.x + h.y) + ((double)l.x + l.y);
    }
};

template <class T> struct Piece {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
    __device__ __forceinline__ float get(int k) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(w[k]);
        } else {
            const unsigned short h = (unsigned short)(w[k / 2] >> (16 * (k % 2)));
            if constexpr (std::is_same<T, __half>::value)
                return __half2float(__ushort_as_half(h));
            else
                return __uint_as_float(k % 2 ? w[k / 2] & 0xFFFF0000u : w[k / 2] << 16);
        }
    }
    // the largest, of a NaN and a number the number
    __device__ __forceinline__ float max(float top) const {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(top, fmaxf(get(0), get(1))), fmaxf(get(2), get(3)));
        } else {
            using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            auto two = [](uint32_t v) { return *reinterpret_cast<const T2 *>(&v); };
            const T2 m = __hmax2(__hmax2(two(raw.x), two(raw.y)), __hmax2(two(raw.z), two(raw.w)));
            return fmaxf(top, fmaxf(to_f32(m.x), to_f32(m.y)));
        }
    }
};

// Where the pieces of a row lie: piece i holds elements i * N - head .. + N - 1.
template <class T> struct RowPieces {
    const T *x;
    int head, vocab, run, first;  // first: this thread's first piece
    __device__ __forceinline__ RowPieces(const T *row, int v) : x(row), vocab(v) {
        head = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
        const int pieces = (v + head + Piece<T>::N - 1) / Piece<T>::N;
        run = (pieces + V_C * V_W * 32 - 1) / (V_C * V_W * 32) * 32;
        first = ((int)cluster_rank() * V_W + (threadIdx.x >> 5)) * run + (threadIdx.x & 31);
    }
    __device__ __forceinline__ int base(int j) const { return place(first + 32 * j); }  // first element of load(j)
    __device__ __forceinline__ int steps() const { return run / 32; }
    __device__ __forceinline__ int place(int piece) const { return piece * Piece<T>::N - head; }  // its first element
    // the j-th piece of this thread
    __device__ __forceinline__ Piece<T> load(int j) const { return at(first + 32 * j); }
    // a piece of the row; what is outside the row is -inf, which weighs nothing
    __device__ __forceinline__ Piece<T> at(int piece) const {
        Piece<T> p;
        const int i = place(piece);
        if (i >= 0 && i + Piece<T>::N <= vocab) {
            p.raw = ld_stream_v4(x + i);
        } else {
            alignas(16) T e[Piece<T>::N];
#pragma unroll
            for (int k = 0; k < Piece<T>::N; k++) e[k] = i + k >= 0 && i + k < vocab ? x[i + k] : from_f32<T>(-INFINITY);
            p.raw = *reinterpret_cast<const uint4 *>(e);
        }
        return p;
    }
};

// Sum of a thread's weights and the first index of the largest logit (greedy), over
// pieces j = 0 .. n - 1 that get(j) gives and base(j) places.
template <class T, class G, class P>
__device__ __forceinline__ void sum_pieces(int n, float top, float inv, bool greedy, G get, P base, double &z, int &arg) {
    constexpr int N = Piece<T>::N;
    if (isfinite(top) && isfinite(inv)) {  // then e^0 is 1 without asking
        const F2 top2 = f2(-top, -top), inv2 = f2(inv, inv);
        Sum01 s;
#pragma unroll
        for (int j = 0; j < n; j++) {
            const Piece<T> p = get(j);
#pragma unroll
            for (int k = 0; k < N; k += 2) {
                const float2 x = split((f2(p.get(k), p.get(k + 1)) + top2) * inv2);
                s.add(f2(fmaxf(expf(x.x), 0.0f), fmaxf(expf(x.y), 0.0f)));  // the maximum drops a NaN
            }
        }
        z += s.get();
    } else {  // nothing above -inf, an infinite logit, a temperature without a finite inverse
#pragma unroll
        for (int j = 0; j < n; j++) {
            const Piece<T> p = get(j);
#pragma unroll
            for (int k = 0; k < N; k++) z += weight(p.get(k), top, inv);
        }
    }
    if (greedy && top > -INFINITY) {
#pragma unroll
        for (int j = 0; j < n; j++) {
            const Piece<T> p = get(j);
#pragma unroll
            for (int k = 0; k < N; k++)
                if (p.get(k) == top) arg = min(arg, base(j) + k);
        }
    }
}

// ---- many logits: two passes -----------------------------------------------------------
// A CTA takes V_CH pieces of a row for the row's largest logit, then (in a second
// kernel) the same pieces for the sum: the weights need the largest of the whole row,
// and reading again, mostly from the L2 cache, costs less than a cluster's meeting for
// it once rows take turns on the SMs. 366 rows of 129,281 bf16: the maxima 18 us (5.2
// TB/s), the sums 46 (issue slots 75 % used), bound by about 25 instructions per
// logit, most of them e^x.
constexpr int V_CH = 1024, V_CT = 256;

template <class T> __global__ void __launch_bounds__(V_CT) k_verify_max(VerifyArgs a) {
    __shared__ float s_top[V_CT / 32];
    pdl_trigger_();
    const int r = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RowPieces<T> row(static_cast<const T *>(a.logits) + r * a.logits_stride, a.vocab);
    Piece<T> p[V_CH / V_CT];
#pragma unroll
    for (int j = 0; j < V_CH / V_CT; j++) p[j] = row.at(blockIdx.x * V_CH + j * V_CT + tid);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < V_CH / V_CT; j++) top = p[j].max(top);
    top = warp_max(top);
    if (lane == 0) s_top[warp] = top;
    __syncthreads();
    if (warp == 0) {
        top = warp_max(lane < V_CT / 32 ? s_top[lane] : -INFINITY);
        if (lane == 0) a.stat[(size_t)r * a.parts + blockIdx.x].top = top;
    }
}

template <class T> __global__ void __launch_bounds__(V_CT) k_verify_sum(VerifyArgs a) {
    __shared__ double s_z[V_CT / 32];
    __shared__ int s_arg[V_CT / 32];
    pdl_trigger_();
    const int r = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RowPieces<T> row(static_cast<const T *>(a.logits) + r * a.logits_stride, a.vocab);
    Piece<T> p[V_CH / V_CT];
#pragma unroll
    for (int j = 0; j < V_CH / V_CT; j++) p[j] = row.at(blockIdx.x * V_CH + j * V_CT + tid);
    const float temp = temp_of(a, seq_of(a, r));
    pdl_wait_();
    RowPart *parts = a.stat + (size_t)r * a.parts;
    float top = -INFINITY;
    for (int i = lane; i < a.parts; i += 32) top = fmaxf(top, __ldcg(&parts[i].top));
    top = warp_max(top);
    double z = 0.0;
    int arg = 0x7FFFFFFF;
    sum_pieces<T>(V_CH / V_CT, top, inv_temp(temp), temp <= 0.0f, [&](int j) { return p[j]; },
                  [&](int j) { return row.place(blockIdx.x * V_CH + j * V_CT + tid); }, z, arg);
    z = warp_sum_d(z);
    arg = __reduce_min_sync(0xffffffffu, arg);
    if (lane == 0) {
        s_z[warp] = z;
        s_arg[warp] = arg;
    }
    __syncthreads();
    if (tid == 0) {
        z = 0.0;
        for (int w = 0; w < V_CT / 32; w++) {
            z += s_z[w];
            arg = min(arg, s_arg[w]);
        }
        parts[blockIdx.x].z = z;
        parts[blockIdx.x].arg = arg;
    }
}

// ---- few rows: one launch, a cluster per row --------------------------------------------
// The largest logit, then every CTA's sum of the weights, from registers (the parts
// meet in row_stat, so the cluster meets once, for the maximum). Bound by issuing
// about 25 instructions per logit, most of them e^x, and by that meeting: 5 greedy rows
// of 32,000 f32, the whole call 6.1 us.
template <class T> __global__ void __cluster_dims__(V_C, 1, 1) __launch_bounds__(V_T, sizeof(T) == 4 ? 2 : 3) k_verify_rows(VerifyArgs a) {
    __shared__ float s_best[V_W], s_cta;
    __shared__ double s_sum[V_W];
    __shared__ int s_arg;
    constexpr int V_NV = v_nv<T>(), N = Piece<T>::N;
    pdl_trigger_();
    const int r = blockIdx.x / V_C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RowPieces<T> row(static_cast<const T *>(a.logits) + r * a.logits_stride, a.vocab);
    Piece<T> keep[V_NV];
    const int steps = row.steps();
#pragma unroll
    for (int j = 0; j < V_NV; j++)
        if (j < steps) keep[j] = row.load(j);
    const float temp = temp_of(a, seq_of(a, r)), inv = inv_temp(temp);
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < V_NV; j++)
        if (j < steps) top = keep[j].max(top);
    for (int j = V_NV; j < steps; j++) top = row.load(j).max(top);
    top = warp_max(top);
    if (lane == 0) s_best[warp] = top;
    if (tid == 0) s_arg = 0x7FFFFFFF;
    __syncthreads();
    if (warp == 0) {
        top = warp_max(lane < V_W ? s_best[lane] : -INFINITY);
        if (lane == 0) s_cta = top;
    }
    cluster_sync();
    top = warp_max(peer_ldf(peer(&s_cta, lane % V_C)));
    cluster_arrive();  // a peer leaves once all have read its shared memory
    double z = 0.0;
    int arg = 0x7FFFFFFF;
    const bool greedy = temp <= 0.0f;
    if (steps >= V_NV) {
        sum_pieces<T>(V_NV, top, inv, greedy, [&](int j) { return keep[j]; }, [&](int j) { return row.base(j); }, z, arg);
    } else {
#pragma unroll
        for (int j = 0; j < V_NV; j++)
            if (j < steps)
                sum_pieces<T>(1, top, inv, greedy, [&](int) { return keep[j]; }, [&](int) { return row.base(j); }, z, arg);
    }
    for (int j = V_NV; j < steps; j++)
        sum_pieces<T>(1, top, inv, greedy, [&](int) { return row.load(j); }, [&](int) { return row.base(j); }, z, arg);
    if (arg != 0x7FFFFFFF) atomicMin(&s_arg, arg);
    z = warp_sum_d(z);
    if (lane == 0) s_sum[warp] = z;
    __syncthreads();
    if (tid == 0) {
        z = 0.0;
#pragma unroll
        for (int w = 0; w < V_W; w++) z += s_sum[w];
        a.stat[r * V_C + cluster_rank()] = RowPart{z, top, s_arg};
    }
    cluster_wait();
}

// One cluster per sequence: the accepted drafts, then one token. The sums of the
// weights over the runs of all the warps say in whose run the chosen index lies, that
// warp's sums over its steps in which of them; it weighs that step again and finds the
// index. Bound by the chain of such meetings and by reading the row: 32 sequences,
// 151,936 f32 logits and probabilities, 29 us cold.
// Without a drafter's probabilities nothing needs the whole row and one CTA does it (C = 1):
// 59 against 65 us for 64 sequences, 366 rows of 129,281 bf16 logits.
template <class T, int C> __global__ void __cluster_dims__(C, 1, 1) __launch_bounds__(V_T, 2) k_verify_pick(VerifyArgs a) {
    __shared__ double s_sum[V_W], s_all[V_C * V_W];
    __shared__ RowStat s_stat[V_W];
    __shared__ bool s_no[V_W];
    constexpr int N = Piece<T>::N;
    const int b = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rank = cluster_rank();
    pdl_wait_();
    const int r0 = (int)min(a.seq_rows[b], (uint32_t)a.n_rows), r1 = (int)min(a.seq_rows[b + 1], (uint32_t)a.n_rows);
    if (r0 >= r1) {  // the whole cluster leaves
        if (tid == 0 && rank == 0) a.n_out[b] = 0;
        return;
    }
    const float t = temp_of(a, b), inv = inv_temp(t);
    const bool greedy = t <= 0.0f;
    auto row_at = [&](int r) { return static_cast<const T *>(a.logits) + r * a.logits_stride; };
    auto logp = [&](const RowStat &s, int r, int tok) {
        if (s.z == 0.0f) return -INFINITY;  // a row with nothing above -inf
        const float l = to_f32(row_at(r)[tok]);
        return fsub(l == s.top ? 0.0f : fmul(fsub(l, s.top), inv), logf(s.z));
    };
    // the first refusal: one row per warp, sixteen at a time
    RowStat s{};
    int stop = r1 - 1;
    for (int j0 = r0; j0 < r1; j0 += V_W) {
        const int r = j0 + warp;
        if (r < r1) {
            const RowStat mine = row_stat(a, r);
            if (lane == 0) {
                bool no = true;  // the last row ends the search too
                if (r < r1 - 1) {
                    const int d = a.tokens[r + 1];
                    if (d >= 0 && d < a.vocab) {
                        if (greedy)
                            no = d != mine.arg;
                        else
                            no = !(fmul(a.u[r], a.probs ? a.probs[r * a.probs_stride + d] : 1.0f) <
                                   __fdiv_rn(weight(to_f32(row_at(r)[d]), mine.top, inv), mine.z));
                        if (rank == 0 && !no) {  // rows after a refusal are written again below
                            a.out[r] = d;
                            a.logprobs[r] = logp(mine, r, d);
                        }
                    }
                }
                s_stat[warp] = mine;
                s_no[warp] = no;
            }
        }
        __syncthreads();
        const uint32_t m = __ballot_sync(0xffffffffu, lane < V_W && j0 + lane < r1 && s_no[lane % V_W]);
        if (m) {
            stop = j0 + __ffs(m) - 1;
            s = s_stat[__ffs(m) - 1];
            break;
        }
        __syncthreads();
    }
    if (rank == 0)
        for (int r = stop + 1 + tid; r < r1; r += V_T) {
            a.out[r] = -1;
            a.logprobs[r] = 0.0f;
        }
    auto emit = [&](int tok) {
        a.out[stop] = tok;
        a.logprobs[stop] = logp(s, stop, tok);
        a.n_out[b] = stop - r0 + 1;
    };
    if (greedy) {
        if (tid == 0 && rank == 0) emit(s.arg);
        return;
    }
    const bool full = stop == r1 - 1;
    const RowPieces<T> row(row_at(stop), a.vocab);
    const float *q = !full && a.probs ? a.probs + stop * a.probs_stride : nullptr;
    const int d = full ? -1 : a.tokens[stop + 1];
    // The weights of the N elements from i on: max(p - q, 0), or without probabilities
    // those of every token but the draft; after the last draft, and when that rest is
    // empty, the target's own.
    bool rest = !full;
    const bool wide = q && (reinterpret_cast<uintptr_t>(q - row.head) & 15) == 0;  // a piece's q in 16 bytes too
    auto load_q = [&](float (&v)[N], int i) {
        if (!rest || !q) return;
        if (wide && i >= 0 && i + N <= a.vocab) {
#pragma unroll
            for (int k = 0; k < N; k += 4) {
                const float4 f = __ldg(reinterpret_cast<const float4 *>(q + i + k));
                v[k] = f.x, v[k + 1] = f.y, v[k + 2] = f.z, v[k + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = i + k >= 0 && i + k < a.vocab ? __ldg(q + i + k) : 0.0f;
        }
    };
    auto weigh = [&](float (&w)[N], const Piece<T> &p, const float (&v)[N], int i) {
#pragma unroll
        for (int k = 0; k < N; k++) w[k] = weight(p.get(k), s.top, inv);
        if (!rest) return;
        if (!q) {
#pragma unroll
            for (int k = 0; k < N; k++)
                if (i + k == d) w[k] = 0.0f;
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) w[k] = fmaxf(fsub(__fdiv_rn(w[k], s.z), v[k]), 0.0f);  // of a NaN, 0
        }
    };
    constexpr int BATCH = sizeof(T) == 4 ? 4 : 2;
    // The cluster goes through the whole row only for max(p - q, 0). Other weights have
    // been summed over the row's parts already (the draft's part again, without it), so
    // one CTA finds the part, and its warps take that.
    const bool whole = C > 1 && q != nullptr;
    if (!whole && rank != 0) return;
    const int per = a.two ? V_CH : V_W * row.run;  // pieces of a part
    int first = row.first, run = row.run, me = (int)rank * V_W + warp;
    double origin = 0.0, want = 0.0;  // sum before the pieces that are gone through, threshold
    auto sum_of = [&](int from, int steps, double &slot, int span) {  // of this warp's steps; a slot of them per lane
        double mine = 0.0;
        slot = 0.0;
        for (int j0 = 0; j0 < steps; j0 += BATCH) {
            Piece<T> p[BATCH];
            float v[BATCH][N];
#pragma unroll
            for (int j = 0; j < BATCH; j++) {  // past the run: past the row, or unused
                p[j] = row.at(from + 32 * (j0 + j));
                load_q(v[j], row.place(from + 32 * (j0 + j)));
            }
#pragma unroll
            for (int j = 0; j < BATCH; j++) {
                if (j0 + j >= steps) break;
                float w[N];
                weigh(w, p[j], v[j], row.place(from + 32 * (j0 + j)));
                Sum01 sum;
#pragma unroll
                for (int k = 0; k < N; k += 2) sum.add(f2(w[k], w[k + 1]));
                const double all = warp_sum_d(sum.get());
                mine += all;
                if ((j0 + j) / span == lane) slot += all;
            }
        }
        return mine;
    };
    if (!whole) {
        const RowPart *parts = a.stat + (size_t)stop * a.parts;
        run = per / V_W;
        int drafts = -1;  // the draft's part
        double dz = 0.0, unused;
        if (rest && d >= 0 && d < a.vocab) {
            drafts = (d + row.head) / N / per;
            const double mine = sum_of(drafts * per + warp * run + lane, run / 32, unused, 1);
            if (lane == 0) s_sum[warp] = mine;
            __syncthreads();
            for (int k = 0; k < V_W; k++) dz += s_sum[k];
            __syncthreads();
        }
        auto z_of = [&](int i) { return i >= a.parts ? 0.0 : i == drafts ? dz : parts[i].z; };
        double total = 0.0;
        for (int pass = 0; pass < 2; pass++) {  // the second when the rest is empty
            total = 0.0;
            for (int i = 0; i < a.parts; i += 32) total += __shfl_sync(0xffffffffu, running(z_of(i + lane)), 31);
            if (total > 0.0 || !rest) break;
            rest = false;
            drafts = -1;
        }
        want = (double)a.u[r1 - 1] * total;
        // the first part whose end exceeds the threshold; the last with weight, should none
        // (a random number of 1), and then the last in it
        int part = -1;
        bool passed = false;
        double at = 0.0;
        for (int i = 0; i < a.parts; i += 32) {
            const double z = z_of(i + lane), end = at + running(z);
            const uint32_t over = __ballot_sync(0xffffffffu, z > 0.0 && end > want), some = __ballot_sync(0xffffffffu, z > 0.0);
            if (over || some) {
                const int l = over ? __ffs(over) - 1 : 31 - __clz(some);
                part = i + l;
                origin = __shfl_sync(0xffffffffu, end - z, l);
            }
            if (over) {
                passed = true;
                break;
            }
            at = __shfl_sync(0xffffffffu, end, 31);
        }
        if (!passed) want = INFINITY;
        if (part < 0) {  // no weight at all
            if (tid == 0) emit(0);
            return;
        }
        first = part * per + warp * run + lane;
        me = warp;
    }
    const int steps = run / 32, span = (steps + 31) / 32;
    double slot = 0.0;  // sum of this warp's steps span lane .. span (lane + 1) - 1
    double upto = 0.0;  // of the sums of warps 4 lane .. 4 lane + 3
    for (int pass = 0; pass < 2; pass++) {  // the second when the rest is empty
        const double mine = sum_of(first, steps, slot, span);
        if (lane == 0) s_sum[warp] = mine;
        if (whole) {
            cluster_sync();
            if (tid < V_C * V_W) s_all[tid] = peer_ldd(peer(&s_sum[tid % V_W], tid / V_W));
            cluster_sync();
        } else {
            __syncthreads();
            if (tid < V_C * V_W) s_all[tid] = tid < V_W ? s_sum[tid] : 0.0;
            __syncthreads();
        }
        double four = 0.0;
#pragma unroll
        for (int k = 0; k < 4; k++) four += s_all[4 * lane + k];
        upto = running(four);
        if (!whole) break;
        const double total = __shfl_sync(0xffffffffu, upto, 31);
        want = (double)a.u[r1 - 1] * total;
        if (total > 0.0 || !rest) break;
        rest = false;
    }
    // the run with the chosen index: the first whose end exceeds the threshold; the
    // last one with weight, should none (a random number of 1, or a part whose sum came
    // out a rounding larger than its runs' together), and in it the last index with weight
    double c = __shfl_up_sync(0xffffffffu, upto, 1), before = 0.0;
    c = lane == 0 ? origin : origin + c;
    int pick = -1, heavy = -1;
    double start = 0.0;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const double v = s_all[4 * lane + k];
        if (v > 0.0) heavy = 4 * lane + k;
        if (pick < 0 && v > 0.0 && c + v > want) {
            pick = 4 * lane + k;
            start = c;
        }
        c += v;
    }
    uint32_t m = __ballot_sync(0xffffffffu, pick >= 0);
    if (m) {
        pick = __shfl_sync(0xffffffffu, pick, __ffs(m) - 1);
        before = __shfl_sync(0xffffffffu, start, __ffs(m) - 1);
    } else {
        pick = __reduce_max_sync(0xffffffffu, heavy);
        want = INFINITY;
    }
    if (pick < 0) {  // no weight at all
        if (tid == 0 && rank == 0) emit(0);
        return;
    }
    if (pick != me) return;
    // the same among the run's slots of steps, then step by step within the slot
    const double ends = before + running(slot);
    m = __ballot_sync(0xffffffffu, slot > 0.0 && ends > want);
    const uint32_t some = __ballot_sync(0xffffffffu, slot > 0.0);
    const int at = m ? __ffs(m) - 1 : 31 - __clz(some);
    before = __shfl_sync(0xffffffffu, ends - slot, at);
    int found = -1, last = -1;
    for (int j = at * span; j < min((at + 1) * span, steps) && found < 0; j++) {
        const int i = row.place(first + 32 * j);
        const Piece<T> p = row.at(first + 32 * j);
        float v[N], e[N];
        load_q(v, i);
        weigh(e, p, v, i);
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < N; k++) sum += e[k];
        const double ends_at = running(sum);
        double here = before + (ends_at - sum);
        before += __shfl_sync(0xffffffffu, ends_at, 31);
        int mine = 0x7FFFFFFF;
#pragma unroll
        for (int k = 0; k < N; k++) {
            here += e[k];
            if (e[k] > 0.0f) {
                last = max(last, i + k);
                if (here > want) mine = min(mine, i + k);
            }
        }
        mine = __reduce_min_sync(0xffffffffu, mine);
        if (mine != 0x7FFFFFFF) found = mine;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 0) emit(found >= 0 ? found : max(last, 0));
}

const char *check(const loom_verify_desc *d) {
    if (!d) return "verify: no descriptor";
    if (!elem_bytes(d->type)) return "verify: type must be LOOM_F32, LOOM_F16 or LOOM_BF16";
    if (!d->vocab || d->vocab > (1u << 24)) return "verify: vocab must be 1..2^24";
    if (d->n_rows > (1u << 24) || d->n_seqs > (1u << 24)) return "verify: at most 2^24 rows and sequences";
    return nullptr;
}

// Two passes, or a cluster per row. On the device the passes are the faster way almost
// from the start (us of a call with probabilities, cluster and passes: f32, 32,000
// logits, 4 rows 11.9 and 11.5, 21 rows 13.8 and 12.5, 36 rows, more clusters than the
// GPU holds at once, 18.2 and 13.0, 169 rows 42 and 25; 1 row of 151,936 16.3 and 10.4;
// bf16, 36 rows of 8,000, 17.1 and 13.3), but their third launch costs the host 2.4 us,
// which decides for calls shorter than the host's part of them.
bool two_passes(const loom_verify_desc *d) {
    const size_t row = d->vocab * elem_bytes(d->type);
    return (d->n_rows * row > ((size_t)5 << 20) || d->n_rows > 32 || row > ((size_t)400 << 10)) && d->n_rows <= 65535;
}
// CTAs to a row: those of its cluster, or of the two passes
int parts_of(const loom_verify_desc *d) {
    if (!two_passes(d)) return V_C;
    const size_t piece = 16 / elem_bytes(d->type), per = V_CH * piece;
    return (int)((d->vocab + piece - 1 + per - 1) / per);  // a row may start inside a piece
}
size_t ws_bytes_of(const loom_verify_desc *d) { return d->n_rows * (size_t)parts_of(d) * sizeof(RowPart); }

template <class T> cudaError_t launch(const VerifyArgs &a, bool two, cudaStream_t st) {
    cudaError_t e;
    if (two) {
        const dim3 grid(a.parts, a.n_rows);
        k_verify_max<T><<<grid, V_CT, 0, st>>>(a);
        count_launch();
        if ((e = cudaGetLastError()) == cudaSuccess) e = launch_pdl_(k_verify_sum<T>, grid, dim3(V_CT), 0, st, a);
    } else {
        k_verify_rows<T><<<(unsigned)a.n_rows * V_C, V_T, 0, st>>>(a);
        count_launch();
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
    return a.probs ? launch_pdl_(k_verify_pick<T, V_C>, dim3((unsigned)a.n_seqs * V_C), dim3(V_T), 0, st, a)
                   : launch_pdl_(k_verify_pick<T, 1>, dim3((unsigned)a.n_seqs), dim3(V_T), 0, st, a);
}

}  // namespace
}  // namespace loom

using namespace loom;

extern "C" {

size_t loom_cuda_verify_workspace(const loom_verify_desc *d) { return check(d) ? 0 : ws_bytes_of(d); }

int loom_cuda_verify(const loom_verify_desc *d, const void *d_logits, const float *d_draft_probs,
                     const int32_t *d_tokens, const uint32_t *d_seq_rows, const float *d_u, const float *d_temperature,
                     int32_t *d_out, int32_t *d_n_out, float *d_logprobs, void *d_ws, size_t ws_bytes, void *stream) {
    if (int rc = rt_need_init()) return rc;
    if (const char *why = check(d)) return rt_decline(why);
    if (d->n_seqs == 0) return LOOM_CUDA_OK;
    if (!d_seq_rows || !d_n_out) return rt_decline("verify: seq_rows and n_out are required");
    if (d->n_rows && (!d_logits || !d_tokens || !d_u || !d_out || !d_logprobs))
        return rt_decline("verify: logits, tokens, u, out and logprobs are required");
    if (ws_bytes < ws_bytes_of(d) || (!d_ws && ws_bytes_of(d))) return rt_decline("verify: workspace too small");
    if (reinterpret_cast<uintptr_t>(d_ws) % 16) return rt_decline("verify: workspace not aligned to 16 bytes");
    VerifyArgs a{};
    a.logits = d_logits;
    a.probs = d_draft_probs;
    a.u = d_u;
    a.temp = d_temperature;
    a.tokens = d_tokens;
    a.seq_rows = d_seq_rows;
    a.out = d_out;
    a.n_out = d_n_out;
    a.logprobs = d_logprobs;
    a.stat = static_cast<RowPart *>(d_ws);
    a.logits_stride = (int64_t)d->logits_stride;
    a.probs_stride = (int64_t)d->probs_stride;
    a.n_seqs = (int)d->n_seqs;
    a.n_rows = (int)d->n_rows;
    a.vocab = (int)d->vocab;
    a.parts = parts_of(d);
    a.two = two_passes(d);
    if (!a.n_rows) {  // every sequence is empty
        const cudaError_t e = cudaMemsetAsync(d_n_out, 0, d->n_seqs * sizeof(int32_t), rt_stream(stream));
        return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("verify", e);
    }
    const cudaError_t e = by_type(d->type, [&](auto t) { return launch<decltype(t)>(a, two_passes(d), rt_stream(stream)); });
    return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("verify", e);
}

}  // extern "C"
