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
#include <cfloat>

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
__device__ __forceinline__ void better(float &v, int &i, float v2, int i2) {
    if (v2 > v || (v2 == v && i2 < i)) {
        v = v2;
        i = i2;
    }
}

constexpr int V_T = 1024;

// the sequence of row r: the last b with seq_rows[b] <= r
__device__ __forceinline__ int seq_of(const VerifyArgs &a, int r) {
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.seq_rows[mid] <= (uint32_t)r) lo = mid; else hi = mid;
    }
    return lo;
}

// one CTA per row: the largest logit, then the sum of the weights
template <class T> __global__ void __launch_bounds__(V_T) k_verify_rows(VerifyArgs a) {
    __shared__ float sv[32];
    __shared__ int si[32];
    __shared__ double sd[32];
    const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T *x = static_cast<const T *>(a.logits) + r * a.logits_stride;
    float top = -INFINITY;
    int arg = 0x7FFFFFFF;
    for (int i = tid; i < a.vocab; i += V_T) {
        const float v = to_f32(x[i]);
        if (v > top) {
            top = v;
            arg = i;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(top, arg, __shfl_xor_sync(0xffffffffu, top, o), __shfl_xor_sync(0xffffffffu, arg, o));
    if (lane == 0) {
        sv[warp] = top;
        si[warp] = arg;
    }
    __syncthreads();
    top = sv[0];
    arg = si[0];
    for (int w = 1; w < 32; w++) better(top, arg, sv[w], si[w]);
    const float inv = inv_temp(temp_of(a, seq_of(a, r)));
    double z = 0.0;
    for (int i = tid; i < a.vocab; i += V_T) z += weight(to_f32(x[i]), top, inv);
    z = warp_sum_d(z);
    if (lane == 0) sd[warp] = z;
    __syncthreads();
    if (tid == 0) {
        z = 0.0;
        for (int w = 0; w < 32; w++) z += sd[w];
        a.stat[r] = RowStat{top, (float)z, arg == 0x7FFFFFFF ? 0 : arg, 0};
    }
}

// one CTA per sequence: the accepted drafts, then one token
template <class T> __global__ void __launch_bounds__(V_T) k_verify_pick(VerifyArgs a) {
    __shared__ double sd[32];
    __shared__ int s_first, s_last, s_stop;
    const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = (int)min(a.seq_rows[b], (uint32_t)a.n_rows), r1 = (int)min(a.seq_rows[b + 1], (uint32_t)a.n_rows);
    if (r0 >= r1) {
        if (tid == 0) a.n_out[b] = 0;
        return;
    }
    const float t = temp_of(a, b), inv = inv_temp(t);
    const bool greedy = t <= 0.0f;
    auto row = [&](int r) { return static_cast<const T *>(a.logits) + r * a.logits_stride; };
    auto logp = [&](int r, int tok) {
        const RowStat s = a.stat[r];
        if (s.z == 0.0f) return -INFINITY;  // a row with nothing above -inf
        const float l = to_f32(row(r)[tok]);
        return fsub(l == s.top ? 0.0f : fmul(fsub(l, s.top), inv), logf(s.z));
    };
    if (tid == 0) {
        int r = r0;
        for (; r < r1 - 1; r++) {
            const int d = a.tokens[r + 1];
            if (d < 0 || d >= a.vocab) break;
            const RowStat s = a.stat[r];
            if (greedy ? d != s.arg
                       : !(fmul(a.u[r], a.probs ? a.probs[r * a.probs_stride + d] : 1.0f) <
                           __fdiv_rn(weight(to_f32(row(r)[d]), s.top, inv), s.z)))
                break;
            a.out[r] = d;
            a.logprobs[r] = logp(r, d);
        }
        s_stop = r;
        s_first = a.vocab;
        s_last = -1;
    }
    __syncthreads();
    const int stop = s_stop;
    const RowStat s = a.stat[stop];
    int tok = s.arg;
    if (!greedy) {
        const T *x = row(stop);
        const bool full = stop == r1 - 1;
        const float *q = a.probs ? a.probs + stop * a.probs_stride : nullptr;
        const int d = full ? -1 : a.tokens[stop + 1];
        const int per = (a.vocab + V_T - 1) / V_T, i0 = min(tid * per, a.vocab), i1 = min(i0 + per, a.vocab);
        double before = 0.0, total = 0.0, mine = 0.0;
        bool rest = !full;
        auto w_at = [&](int i) {
            const float e = weight(to_f32(x[i]), s.top, inv);
            if (!rest) return e;
            if (!q) return i == d ? 0.0f : e;
            const float left = fsub(__fdiv_rn(e, s.z), q[i]);
            return left > 0.0f ? left : 0.0f;
        };
        for (int pass = 0; pass < 2; pass++) {  // the second when the rest is empty: from p
            mine = 0.0;
            for (int i = i0; i < i1; i++) mine += w_at(i);
            double run = mine;  // running sum over the threads, each with its run of the vocabulary
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double v = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += v;
            }
            __syncthreads();
            if (lane == 31) sd[warp] = run;
            __syncthreads();
            before = run - mine;
            total = 0.0;
            for (int w = 0; w < 32; w++) {
                if (w < warp) before += sd[w];
                total += sd[w];
            }
            if (total > 0.0 || !rest) break;
            rest = false;
        }
        const double want = (double)a.u[r1 - 1] * total;
        int first = a.vocab, last = -1;
        double c = before;
        for (int i = i0; i < i1; i++) {
            const float w = w_at(i);
            c += w;
            if (w > 0.0f) {
                last = i;
                if (c > want && first == a.vocab) first = i;
            }
        }
        if (first < a.vocab) atomicMin(&s_first, first);
        if (last >= 0) atomicMax(&s_last, last);
        __syncthreads();
        tok = s_first < a.vocab ? s_first : s_last >= 0 ? s_last : 0;
    }
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
    k_verify_rows<T><<<a.n_rows, V_T, 0, st>>>(a);
    k_verify_pick<T><<<a.n_seqs, V_T, 0, st>>>(a);
    count_launches(2);
    return cudaGetLastError();
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
