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

struct RowStat {
    float top;     // largest logit that is not NaN; -inf when none is above it
    float z;       // sum of e^((l - top) / T)
    int arg;       // its first index
    int pad;
};

struct VerifyArgs {
    const void *logits;
    const float *probs, *u, *temp;
    const int32_t *tokens;
    const uint32_t *seq_rows;
    int32_t *out, *n_out;
    float *logprobs;
    RowStat *stat;
    int64_t logits_stride, probs_stride;
    int n_seqs, n_rows, vocab;
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

// ---- layout of a row over a cluster -----------------------------------------------
// A row of logits is spread over a cluster of V_C CTAs of V_W warps: warp k of the
// cluster's V_C * V_W has the k-th run of `run` 16-byte pieces, its lane l the
// pieces l, l + 32, ... of the run. So a running sum over the vocabulary is one
// over the warps, then over groups of 32 pieces, then over lanes. A thread keeps
// its first v_nv pieces in registers (152,000 f32 logits take 9.3 of them), so the
// row crosses the memory once although the weights need its maximum; longer rows
// read the rest again. A row that does not start on 16 bytes is shifted: its first
// piece holds fewer logits.
constexpr int V_C = 8, V_W = 16, V_T = V_W * 32;
template <class T> constexpr int v_nv() { return sizeof(T) == 4 ? 10 : 5; }

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address in CTA `rank` of a variable of this CTA's shared memory
__device__ __forceinline__ uint32_t peer(const void *p, unsigned rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ uint64_t peer_ld(uint32_t a) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}

__device__ __forceinline__ int peer_ld32(uint32_t a) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

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
                return __bfloat162float(__ushort_as_bfloat16(h));
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
    __device__ __forceinline__ int base(int j) const { return (first + 32 * j) * Piece<T>::N - head; }  // element
    __device__ __forceinline__ int steps() const { return run / 32; }
    // the j-th piece of this thread; outside the row -inf, which weighs nothing
    __device__ __forceinline__ Piece<T> load(int j) const {
        Piece<T> p;
        const int i = base(j);
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

// One cluster per row: the largest logit and its first index, then the sum of the
// weights. Bound by reading the logits once.
template <class T> __global__ void __cluster_dims__(V_C, 1, 1) __launch_bounds__(V_T, 2) k_verify_rows(VerifyArgs a) {
    __shared__ uint64_t s_best[V_W], s_cta;
    __shared__ double s_sum[V_W], s_z;
    constexpr int V_NV = v_nv<T>();
    pdl_trigger_();
    const int r = blockIdx.x / V_C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RowPieces<T> row(static_cast<const T *>(a.logits) + r * a.logits_stride, a.vocab);
    const float inv = inv_temp(temp_of(a, seq_of(a, r)));
    Piece<T> keep[V_NV];
    const int steps = row.steps();
#pragma unroll
    for (int j = 0; j < V_NV; j++)
        if (j < steps) keep[j] = row.load(j);
    // the best of (logit, lowest index) as one number: order-preserving bits of the
    // logit above the complement of the index
    float top = -INFINITY;
    int arg = -1;
    auto look = [&](const Piece<T> &p, int j) {
#pragma unroll
        for (int k = 0; k < Piece<T>::N; k++) {
            const float v = p.get(k);
            if (v > top) {
                top = v;
                arg = row.base(j) + k;
            }
        }
    };
#pragma unroll
    for (int j = 0; j < V_NV; j++)
        if (j < steps) look(keep[j], j);
    for (int j = V_NV; j < steps; j++) look(row.load(j), j);
    const uint32_t bits = __float_as_uint(top + 0.0f);  // -0 and 0 are equal
    uint64_t best = arg < 0 ? 0 : ((uint64_t)(bits & 0x80000000u ? ~bits : bits | 0x80000000u) << 32) | (uint32_t)~arg;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, (uint64_t)__shfl_xor_sync(0xffffffffu, (unsigned long long)best, o));
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    best = s_best[0];
    for (int w = 1; w < V_W; w++) best = max(best, s_best[w]);
    if (tid == 0) s_cta = best;
    cluster_sync();
    for (unsigned c = 0; c < V_C; c++) best = max(best, peer_ld(peer(&s_cta, c)));
    const uint32_t hi = (uint32_t)(best >> 32);
    top = best ? __uint_as_float(hi & 0x80000000u ? hi & 0x7FFFFFFFu : ~hi) : -INFINITY;
    double z = 0.0;
    auto add = [&](const Piece<T> &p) {
#pragma unroll
        for (int k = 0; k < Piece<T>::N; k++) z += weight(p.get(k), top, inv);
    };
#pragma unroll
    for (int j = 0; j < V_NV; j++)
        if (j < steps) add(keep[j]);
    for (int j = V_NV; j < steps; j++) add(row.load(j));
    z = warp_sum_d(z);
    if (lane == 0) s_sum[warp] = z;
    __syncthreads();
    if (tid == 0) {
        z = 0.0;
        for (int w = 0; w < V_W; w++) z += s_sum[w];
        s_z = z;
    }
    cluster_sync();
    if (tid == 0 && cluster_rank() == 0) {
        z = 0.0;
        for (unsigned c = 0; c < V_C; c++) z += __longlong_as_double((long long)peer_ld(peer(&s_z, c)));
        a.stat[r] = RowStat{top, (float)z, best ? (int)~(uint32_t)best : 0, 0};
    }
    cluster_sync();  // the others' shared memory is being read
}

// One cluster per sequence: the accepted drafts, then one token. The weights of the
// row at the refusal are kept in registers while their sums say in which warp's run,
// which group of 32 pieces and which lane the chosen index lies.
template <class T> __global__ void __cluster_dims__(V_C, 1, 1) __launch_bounds__(V_T, 1) k_verify_pick(VerifyArgs a) {
    __shared__ double s_sum[V_W], s_cta;
    __shared__ int s_stop, s_first, s_last;
    constexpr int V_NV = v_nv<T>();
    const int b = blockIdx.x / V_C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
    auto logp = [&](int r, int tok) {
        const RowStat s = a.stat[r];
        if (s.z == 0.0f) return -INFINITY;  // a row with nothing above -inf
        const float l = to_f32(row_at(r)[tok]);
        return fsub(l == s.top ? 0.0f : fmul(fsub(l, s.top), inv), logf(s.z));
    };
    // the first refusal: one draft per lane of the first warp
    if (warp == 0) {
        int stop = r1 - 1;
        for (int j = r0; j < r1 - 1; j += 32) {
            const int r = j + lane;
            bool no = false;
            if (r < r1 - 1) {
                const int d = a.tokens[r + 1];
                const RowStat s = a.stat[r];
                if (d < 0 || d >= a.vocab)
                    no = true;
                else if (greedy)
                    no = d != s.arg;
                else
                    no = !(fmul(a.u[r], a.probs ? a.probs[r * a.probs_stride + d] : 1.0f) <
                           __fdiv_rn(weight(to_f32(row_at(r)[d]), s.top, inv), s.z));
                if (rank == 0 && !no) {  // a row after a refusal is written again below
                    a.out[r] = d;
                    a.logprobs[r] = logp(r, d);
                }
            }
            const uint32_t m = __ballot_sync(0xffffffffu, no);
            if (m) {
                stop = j + __ffs(m) - 1;
                break;
            }
        }
        if (lane == 0) {
            s_stop = stop;
            s_first = 0x7FFFFFFF;
            s_last = -1;
        }
    }
    __syncthreads();
    const int stop = s_stop;
    const RowStat s = a.stat[stop];
    int tok = s.arg;
    if (!greedy) {
        const bool full = stop == r1 - 1;
        const RowPieces<T> row(row_at(stop), a.vocab);
        const float *q = !full && a.probs ? a.probs + stop * a.probs_stride : nullptr;
        const int d = full ? -1 : a.tokens[stop + 1];
        const int steps = row.steps();
        bool rest = !full;
        // weight of element i with logit l: max(p - q, 0), or without probabilities
        // every token but the draft, or (after the last draft, or when the rest is
        // empty) the target's own
        auto w_of = [&](float l, int i) {
            const float e = weight(l, s.top, inv);
            if (!rest || i < 0 || i >= a.vocab) return e;
            if (!q) return i == d ? 0.0f : e;
            const float left = fsub(__fdiv_rn(e, s.z), __ldg(q + i));
            return left > 0.0f ? left : 0.0f;
        };
        constexpr int N = Piece<T>::N;
        float w[V_NV][N];
        double mine = 0.0, total = 0.0, before = 0.0;
        for (int pass = 0; pass < 2; pass++) {  // the second when the rest is empty
            mine = 0.0;
#pragma unroll
            for (int j = 0; j < V_NV; j++)
                if (j < steps) {
                    const Piece<T> p = row.load(j);
#pragma unroll
                    for (int k = 0; k < N; k++) mine += w[j][k] = w_of(p.get(k), row.base(j) + k);
                }
            for (int j = V_NV; j < steps; j++) {
                const Piece<T> p = row.load(j);
#pragma unroll
                for (int k = 0; k < N; k++) mine += w_of(p.get(k), row.base(j) + k);
            }
            mine = warp_sum_d(mine);
            __syncthreads();
            if (lane == 0) s_sum[warp] = mine;
            __syncthreads();
            if (tid == 0) {
                double c = 0.0;
                for (int k = 0; k < V_W; k++) c += s_sum[k];
                s_cta = c;
            }
            cluster_sync();
            total = before = 0.0;
            for (unsigned c = 0; c < V_C; c++) {
                const double v = __longlong_as_double((long long)peer_ld(peer(&s_cta, c)));
                if (c < rank) before += v;
                total += v;
            }
            for (int k = 0; k < warp; k++) before += s_sum[k];
            cluster_sync();  // s_cta has been read
            if (total > 0.0 || !rest) break;
            rest = false;
        }
        // The first index whose running sum exceeds the threshold, and the last one
        // with any weight, which is taken when rounding leaves no such index.
        const double want = (double)a.u[r1 - 1] * total;
        int first = 0x7FFFFFFF, last = -1;
        if (mine > 0.0) {  // the warp has weight; `before` precedes its run
            double c = before;
            for (int j = 0; j < steps; j++) {
                float e[N];
                if (j < V_NV) {
#pragma unroll
                    for (int jj = 0; jj < V_NV; jj++)
                        if (jj == j) {
#pragma unroll
                            for (int k = 0; k < N; k++) e[k] = w[jj][k];
                        }
                } else {
                    const Piece<T> p = row.load(j);
#pragma unroll
                    for (int k = 0; k < N; k++) e[k] = w_of(p.get(k), row.base(j) + k);
                }
                double sum = 0.0;
#pragma unroll
                for (int k = 0; k < N; k++) sum += e[k];
                double upto = sum;  // over the lanes
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                double run = c + (upto - sum);
#pragma unroll
                for (int k = 0; k < N; k++) {
                    run += e[k];
                    if (e[k] > 0.0f) {
                        last = row.base(j) + k;
                        if (run > want) first = min(first, last);
                    }
                }
                c += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (first != 0x7FFFFFFF) atomicMin(&s_first, first);
        if (last >= 0) atomicMax(&s_last, last);
        cluster_sync();
        int lo = 0x7FFFFFFF, hi = -1;
        for (unsigned c = 0; c < V_C && rank == 0; c++) {
            lo = min(lo, peer_ld32(peer(&s_first, c)));
            hi = max(hi, peer_ld32(peer(&s_last, c)));
        }
        tok = lo != 0x7FFFFFFF ? lo : hi >= 0 ? hi : 0;
        cluster_sync();  // the others' shared memory has been read
    }
    if (rank != 0) return;
    __syncthreads();
    if (tid == 0) {
        a.out[stop] = tok;
        a.logprobs[stop] = logp(stop, tok);
        a.n_out[b] = stop - r0 + 1;
    }
    for (int r = stop + 1 + tid; r < r1; r += V_T) {
        a.out[r] = -1;
        a.logprobs[r] = 0.0f;
    }
}

const char *check(const loom_verify_desc *d) {
    if (!d) return "verify: no descriptor";
    if (!elem_bytes(d->type)) return "verify: type must be LOOM_F32, LOOM_F16 or LOOM_BF16";
    if (!d->vocab || d->vocab > (1u << 24)) return "verify: vocab must be 1..2^24";
    if (d->n_rows > (1u << 24) || d->n_seqs > (1u << 24)) return "verify: at most 2^24 rows and sequences";
    return nullptr;
}

size_t ws_bytes_of(const loom_verify_desc *d) { return d->n_rows * sizeof(RowStat); }

template <class T> cudaError_t launch(const VerifyArgs &a, cudaStream_t st) {
    k_verify_rows<T><<<(unsigned)a.n_rows * V_C, V_T, 0, st>>>(a);
    count_launch();
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? launch_pdl_(k_verify_pick<T>, dim3((unsigned)a.n_seqs * V_C), dim3(V_T), 0, st, a) : e;
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
    a.stat = static_cast<RowStat *>(d_ws);
    a.logits_stride = (int64_t)d->logits_stride;
    a.probs_stride = (int64_t)d->probs_stride;
    a.n_seqs = (int)d->n_seqs;
    a.n_rows = (int)d->n_rows;
    a.vocab = (int)d->vocab;
    if (!a.n_rows) {  // every sequence is empty
        const cudaError_t e = cudaMemsetAsync(d_n_out, 0, d->n_seqs * sizeof(int32_t), rt_stream(stream));
        return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("verify", e);
    }
    const cudaError_t e = by_type(d->type, [&](auto t) { return launch<decltype(t)>(a, rt_stream(stream)); });
    return e == cudaSuccess ? LOOM_CUDA_OK : rt_fail("verify", e);
}

}  // extern "C"
