// attn_prefix.cu -- the shared prefix's part of loom_cuda_attn_shared on the
// 5th-generation tensor cores (attn_shared.cu has the operator).
//
// With many sequences the prefix is a matrix product: every position's keys and
// values (512 bytes of a KV head) meet all the batch's query rows of the head's
// group, so beyond about 100 rows the arithmetic, not the memory, takes the time.
// A CTA has up to 256 query rows (two tiles of 128, the height of an MMA) and a
// chunk of positions, 64 at a time:
//
//   S = Q K^T   both from shared memory, into TMEM (128 lanes = rows, 64 columns)
//   P = 2^(scale S - m)   by the row's thread: maximum, exponentials, sum, P in the
//               element type back into TMEM in S's place
//   O += P V    P from TMEM, V from shared memory as it lies (positions x
//               dimensions: the operand with the summed dimension outermost)
//
// A tile has two S (and a barrier of each kind for each: its threads may be a step
// ahead of the products), so the products of the next positions are made while its
// threads are at their exponentials. A step of two full tiles is 1,024 cycles of products
// and, at 16 an SM and cycle, 1,024 of exponentials; it takes about 2,500 (1.3 us), so
// neither pipe is full (tensor 47 %, issue 36 %): P V of either tile waits for both
// tiles' P, and the next S for that. Steps of 128 positions with one S a tile took 131 to
// 141 us where these take 117, tiles a quarter step apart 125. O
// stays in TMEM; it is scaled when a row's maximum has grown by more than 2^8 over
// the one in use (the quotient by the sum undoes any common factor, and f32 has
// room), so after the first positions hardly ever.
//
// Roles (320 threads, one CTA per SM: all 512 TMEM columns): warps 0-3 and 4-7 the
// rows of tile 0 and 1, warp 8 the copies (TMA, 64 positions of keys or values
// each, through a ring of six 16 KB stages), warp 9 the MMAs. The ring's size and
// 112 registers a thread leave room on the SM for a CTA of the own caches' kernel,
// which is bound by memory where this one is not. P is rounded to the element type
// for its product, as in attn_shared.cu; its sum is taken before that, since with the
// weights as rounded the errors are the same (64 rows over 8,192 positions: 2.3e-3 bf16,
// 2.9e-4 f16) and the call took 166 us, not 162. 192 rows of 8 heads (128 sequences' drafts) over 32,768 positions
// of 4 KV heads of 128, bf16: 103 GFLOP in 109 to 122 us by the clocks, up to 950
// TFLOP/s; 64 sequences' 200 rows over 8,192 positions 47 us. Every wait is bounded; one that gives up sets an error word
// (bit 128 of loom_cuda_device_error), leaves NaN in the CTA's rows and ends.
#include <type_traits>

#include "attn_shared.cuh"

namespace loom {
namespace {

constexpr int AP_THREADS = 320, AP_N = ATTN_PREFIX_N, AP_STAGES = 6;
constexpr size_t AP_QBLOCK = 128 * 128;          // 128 rows of 64 elements, swizzled in 128-byte rows
constexpr size_t AP_BLOCK = AP_N * 128;          // the same of 64 positions
constexpr float AP_LAZY = 8.0f;                  // log2 of the growth that scales O

struct ApBars {
    uint64_t full[AP_STAGES], empty[AP_STAGES], s_full[2][2], p_full[2][2], o_done[2][2];  // [tile][step & 1]
    uint64_t drain;
    uint32_t tmem;
    int err, issued;  // a wait gave up; copies issued
};

__device__ unsigned g_gave_up;  // CTAs of which a wait gave up

template <int NB> constexpr size_t ap_smem() {  // queries of two tiles, the ring, barriers
    return NB * (2 * AP_QBLOCK + AP_STAGES * AP_BLOCK) + sizeof(ApBars);
}

// 128-byte-swizzled tile, the summed dimension along the rows' 128 bytes
__device__ __forceinline__ uint64_t ap_desc_k(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// the same tile with the summed dimension down the rows: 64 columns of 8 rows are an
// atom of 1 KB, the next 8 rows follow (stride offset), the next 64 columns are a
// block further (leading offset)
__device__ __forceinline__ uint64_t ap_desc_mn(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(AP_BLOCK >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// kind::f16, f32 accumulator, M = 128; b_rows: B's summed dimension down its rows
template <class T> __device__ __forceinline__ uint32_t ap_idesc(int n, bool b_rows) {
    const uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)b_rows << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// Products are issued by one lane: the warp runs the issuing loop and its waits as a
// whole and branches on this only around the products, so that the descriptors stay
// in uniform registers (a loop run by one lane alone moves them there before every
// product, which took longer than the product).
__device__ __forceinline__ bool ap_elect() {
    uint32_t q;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(q));
    return q != 0;
}
__device__ __forceinline__ void ap_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    umma_bf16(d, a, b, idesc, acc);
}
__device__ __forceinline__ void ap_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
        : "memory");
}
#define AP_R8(r, o) "=r"(r[o]), "=r"(r[o + 1]), "=r"(r[o + 2]), "=r"(r[o + 3]), "=r"(r[o + 4]), "=r"(r[o + 5]), "=r"(r[o + 6]), "=r"(r[o + 7])
#define AP_I8(r, o) "r"(r[o]), "r"(r[o + 1]), "r"(r[o + 2]), "r"(r[o + 3]), "r"(r[o + 4]), "r"(r[o + 5]), "r"(r[o + 6]), "r"(r[o + 7])
// 32 columns of the warp's lanes, without the wait
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : AP_R8(r, 0), AP_R8(r, 8), AP_R8(r, 16), AP_R8(r, 24)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : AP_R8(r, 0), AP_R8(r, 8)
        : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::AP_I8(r, 0),
        AP_I8(r, 8), "r"(addr)
        : "memory");
}
#define AP_W8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
// the reads so far are done; the registers are named so that no use of them moves above the wait
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : AP_W8(r, 0), AP_W8(r, 8), AP_W8(r, 16), AP_W8(r, 24)::"memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : AP_W8(r, 0), AP_W8(r, 8)::"memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// columns from `left` on are no positions
__device__ __forceinline__ void ap_mask(uint32_t (&s)[32], int left) {
    if (left >= 32) return;
#pragma unroll
    for (int k = 0; k < 32; k++)
        if (k >= left) s[k] = 0xFF800000u;  // -inf
}

// NB: blocks of 64 dimensions (head_dim <= 64 NB)
template <class T, int NB>
__global__ void __maxnreg__(112)
    k_attn_prefix(AttnArgs a, const __grid_constant__ AttnMaps maps) {
    extern __shared__ __align__(1024) uint8_t smp[];  // the swizzle's atoms are 1 KB
    pdl_trigger_();
    const uint32_t sm0 = smem_u32(smp);
    const uint32_t ring = sm0 + 2 * NB * AP_QBLOCK;
    ApBars &B = *reinterpret_cast<ApBars *>(smp + NB * (2 * AP_QBLOCK + AP_STAGES * AP_BLOCK));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, hd = a.hd;
    const Item<T> it = item_of<T>(a, blockIdx.x, kvh);
    const int n = (it.p1 - it.p0 + AP_N - 1) / AP_N, rows = it.r1 - it.r0, tiles = rows > 128 ? 2 : 1;
    volatile int *err = &B.err;
    auto wait = [&](uint64_t *bar, uint32_t parity) {  // false once any wait of the CTA has given up
        for (int i = 0; i < ATTN_LOOKS; i++) {
            if (mbar_wait(bar, parity, ATTN_POLLS)) return true;
            if (*err) return false;
        }
        *err = 1;
        return false;
    };
    // The ring's items in the order of their use: keys 0 and 1, then values j and keys
    // j + 2 for every step j. Item i of the list, of which there are 2 n, is of
    // keys or values of step `pos`.
    auto item_pos = [&](int i, bool &values) {
        const int lead = min(n, 2);
        values = i >= lead && (i - lead < 2 * (n - lead) ? (i - lead) % 2 == 0 : true);
        if (i < lead) return i;
        return i - lead < 2 * (n - lead) ? (i - lead) / 2 + (values ? 0 : lead) : (n - lead) + (i - lead - 2 * (n - lead));
    };
    auto fetch = [&](int i) {
        const int s = i % AP_STAGES;
        bool values;
        const int pos = item_pos(i, values);
        mbar_expect_tx(&B.full[s], (uint32_t)(NB * AP_BLOCK));
        B.issued = i + 1;
        for (int b = 0; b < NB; b++)
            attn_tma(ring + (uint32_t)((s * NB + b) * AP_BLOCK), values ? &maps.pv : &maps.pk, b * 64, it.p0 + pos * AP_N, kvh, 0,
                     &B.full[s]);
    };
    if (warp == 8 && lane == 0) {
        for (int s = 0; s < AP_STAGES; s++) {
            mbar_init_nf(&B.full[s], 1);
            mbar_init_nf(&B.empty[s], 1);
        }
        for (int t = 0; t < 2; t++) {
            for (int b = 0; b < 2; b++) {
                mbar_init_nf(&B.s_full[t][b], 1);
                mbar_init_nf(&B.p_full[t][b], 128);
                mbar_init_nf(&B.o_done[t][b], 1);
            }
        }
        mbar_init_nf(&B.drain, 1);
        B.err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = 0; i < AP_STAGES && i < 2 * n; i++) fetch(i);
    }
    if (warp == 9) tmem_alloc(&B.tmem, 512);
    // queries: 16-byte pieces into the swizzled tiles; zeros past the rows and dimensions
    const bool whole = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.q_stride % 8 == 0;
    for (int i = tid; i < tiles * 128 * NB * 8; i += AP_THREADS) {
        const int j = i / (NB * 8), c = i % (NB * 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (j < rows && c * 8 < hd) {
            const int hr = it.r0 + j;
            const T *src = static_cast<const T *>(a.q) + (int64_t)(hr / a.group) * a.q_stride +
                           (int64_t)(kvh * a.group + hr % a.group) * hd + c * 8;
            if (whole) {
                v = ld_v4(src);
            } else {
                alignas(16) T e[8];
                for (int k = 0; k < 8; k++) e[k] = src[k];
                v = *reinterpret_cast<const uint4 *>(e);
            }
        }
        const int tl = j >> 7, r = j & 127;
        *reinterpret_cast<uint4 *>(smp + (size_t)(tl * NB + c / 8) * AP_QBLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
    }
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = B.tmem;
    if (warp == 8) {
        if (lane == 0)
            for (int i = AP_STAGES; i < 2 * n; i++) {
                if (!wait(&B.empty[i % AP_STAGES], ((i / AP_STAGES) - 1) & 1)) break;
                fetch(i);
            }
        __syncwarp();
    } else if (warp == 9) {
        // 24 products a step. A wait that gives up does not end the loop (its bound
        // holds for all together: after one the others return at once).
        const uint32_t id_s = ap_idesc<T>(AP_N, false), id_o = ap_idesc<T>((hd + 15) / 16 * 16, true);
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
        const int ks = (hd + 15) / 16;
        const uint64_t dq = ap_desc_k(sm0), dk = ap_desc_k(ring), dv = ap_desc_mn(ring);
        constexpr uint32_t STAGE = NB * AP_BLOCK >> 4;  // in the descriptors' 16 bytes
        int st = 0;                                     // the ring's present stage
        uint32_t ph = 0;                                // and its parity
        auto step = [&]() {
            if (++st == AP_STAGES) {
                st = 0;
                ph ^= 1;
            }
        };
        // the tiles' products alternate: one that adds to the result of the one before
        // it waits for that to leave the pipe
        auto qk = [&](int b) {  // S = Q K^T of both tiles, keys in the present stage
            const uint64_t k = dk + (uint32_t)st * STAGE;
            const uint32_t d = tm + b * 64;
            if (!ap_elect()) return;
#pragma unroll
            for (int s = 0; s < NB * 4; s++)
                if (s < ks) {
                    const uint64_t q = dq + ((s >> 2) * (AP_QBLOCK >> 4) + (s & 3) * 2), ks_ = k + ((s >> 2) * (AP_BLOCK >> 4) + (s & 3) * 2);
                    ap_mma_ss(d, q, ks_, id_s, s > 0);
                    if (tiles > 1) ap_mma_ss(d + 128, q + (NB * AP_QBLOCK >> 4), ks_, id_s, s > 0);
                }
            umma_commit(&B.s_full[0][b]);
            if (tiles > 1) umma_commit(&B.s_full[1][b]);
            umma_commit(&B.empty[st]);
        };
        for (int j = 0; j < 2 && j < n; j++) {
            wait(&B.full[st], ph);
            tc_fence_after();
            qk(j);
            step();
        }
        for (int j = 0; j < n; j++) {
            // values j in the present stage, keys j + 2 (if any) in the next
            const int b = j & 1;
            wait(&B.full[st], ph);
            wait(&B.p_full[0][b], (j >> 1) & 1);
            if (tiles > 1) wait(&B.p_full[1][b], (j >> 1) & 1);
            tc_fence_after();
            const uint64_t v = dv + (uint32_t)st * STAGE;
            if (ap_elect()) {
#pragma unroll
                for (int s = 0; s < AP_N / 16; s++) {
                    ap_mma_ts(tm + 256, tm + b * 64 + s * 8, v + s * (2048 >> 4), id_o, j > 0 || s > 0);
                    if (tiles > 1) ap_mma_ts(tm + 384, tm + 128 + b * 64 + s * 8, v + s * (2048 >> 4), id_o, j > 0 || s > 0);
                }
                umma_commit(&B.o_done[0][b]);
                if (tiles > 1) umma_commit(&B.o_done[1][b]);
                umma_commit(&B.empty[st]);
            }
            __syncwarp();
            step();
            if (j + 2 < n) {
                wait(&B.full[st], ph);
                qk(b);
                step();
            }
        }
    } else if (warp / 4 < tiles) {
        const int t = warp / 4, row = it.r0 + t * 128 + (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), ts = lanes + t * 128, to = lanes + 256 + t * 128;
        float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        bool ok = !a.fail;
        if (!ok) *err = 1;
        for (int j = 0; j < n && ok; j++) {
            ok = __all_sync(0xffffffffu, wait(&B.s_full[t][j & 1], (j >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const uint32_t tp = ts + (j & 1) * 64;
            const int left = it.p1 - (it.p0 + j * AP_N);
            uint32_t s[2][32];
            tmem_ld32(tp, s[0]);
            tmem_ld32(tp + 32, s[1]);
            tmem_wait_ld(s[0]);
            tmem_wait_ld(s[1]);
            ap_mask(s[0], left);
            ap_mask(s[1], left - 32);
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < 64; k++) x[k & 3] = fmaxf(x[k & 3], __uint_as_float(s[k / 32][k % 32]));
            const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale;  // scale > 0
            if (__any_sync(0xffffffffu, top > m + AP_LAZY || (m == -INFINITY && top > m))) {
                const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.0f : ex2(m - mn);
                l0 *= f;
                l1 *= f;
                m = mn;
                if (j) {  // the step before is in O, and this one is not: its P is not made
                    ok = __all_sync(0xffffffffu, wait(&B.o_done[t][(j - 1) & 1], ((j - 1) >> 1) & 1));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < NB * 64; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(to + c, o);
                        tmem_wait_ld(o);
#pragma unroll
                        for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_st16(to + c, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                uint32_t p[16];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float e0 = ex2(fmaf(__uint_as_float(s[c][2 * k]), a.scale, -base));
                    const float e1 = ex2(fmaf(__uint_as_float(s[c][2 * k + 1]), a.scale, -base));
                    l0 += e0;
                    l1 += e1;
                    p[k] = pack2<T>(e0, e1);
                }
                tmem_st16(tp + c * 16, p);
            }
            tmem_wait_st();
            tc_fence_before();
            attn_arrive(&B.p_full[t][j & 1]);
        }
        if (ok) ok = __all_sync(0xffffffffu, wait(&B.o_done[t][(n - 1) & 1], ((n - 1) >> 1) & 1));
        if (ok) {
            tc_fence_after();
            const bool in = row < it.r1;
            const size_t at = in ? part_at(a, it.slot, row, kvh) : 0;
            if (in) a.ml[at] = make_float2(m, l0 + l1);
            float *dst = a.acc + at * hd;
            for (int c = 0; c < hd; c += 16) {
                uint32_t o[16];
                tmem_ld16(to + c, o);
                tmem_wait_ld(o);
                if (in)
#pragma unroll
                    for (int k = 0; k < 16; k += 4)
                        if (c + k < hd)  // hd is a multiple of 8
                            *reinterpret_cast<uint4 *>(dst + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (*err) {  // what was issued ends before the memory it uses is given back
        if (warp == 9 && ap_elect()) {  // the lane that issued the products
            umma_commit(&B.drain);
            attn_drain(&B.drain, 0);
            for (int i = max(B.issued - AP_STAGES, 0); i < B.issued; i++) attn_drain(&B.full[i % AP_STAGES], (i / AP_STAGES) & 1);
            atomicAdd(&g_gave_up, 1u);
        }
        for (int j = tid; j < rows; j += AP_THREADS) a.ml[part_at(a, it.slot, it.r0 + j, kvh)] = make_float2(NAN, NAN);
        __syncthreads();
    }
    tc_fence_after();
    if (warp == 9) tmem_free(tmem, 512);
}

template <class T, int NB> cudaError_t ap_launch(const AttnArgs &a, const AttnMaps &maps, cudaStream_t st) {
    if (const cudaError_t e = allow_smem<k_attn_prefix<T, NB>>(ap_smem<NB>()); e != cudaSuccess) return e;
    k_attn_prefix<T, NB><<<dim3(a.n_pre * a.pre_tiles, a.nkv), AP_THREADS, ap_smem<NB>(), st>>>(a, maps);
    count_launch();
    return cudaGetLastError();
}

}  // namespace

cudaError_t attn_prefix_gave_up(unsigned *v, cudaStream_t st) {
    return cudaMemcpyFromSymbolAsync(v, g_gave_up, sizeof *v, 0, cudaMemcpyDeviceToHost, st);
}

cudaError_t attn_prefix_run(int type, const AttnArgs &a, const AttnMaps &maps, cudaStream_t st) {
    if (type == T_F16) return a.hd <= 64 ? ap_launch<__half, 1>(a, maps, st) : ap_launch<__half, 2>(a, maps, st);
    return a.hd <= 64 ? ap_launch<__nv_bfloat16, 1>(a, maps, st) : ap_launch<__nv_bfloat16, 2>(a, maps, st);
}

}  // namespace loom
