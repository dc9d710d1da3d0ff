// attn_prefix.cu -- the shared prefix's part of loom_cuda_attn_shared on the
// 5th-generation tensor cores (attn_shared.cu has the operator).
//
// With many sequences the prefix is a matrix product: every position's keys and
// values (512 bytes of a KV head) meet all the batch's query rows of the head's
// group, so beyond about 100 rows the arithmetic, not the memory, takes the time.
// A CTA has up to 256 query rows (two tiles of 128, the height of an MMA) and a
// chunk of positions, 128 at a time:
//
//   S = Q K^T   both from shared memory, into TMEM (128 lanes = rows, 128 columns)
//   P = 2^(scale S - m)   by the row's thread: maximum, exponentials, sum, P in the
//               element type back into TMEM in S's place
//   O += P V    P from TMEM, V from shared memory as it lies (positions x
//               dimensions: the operand with the summed dimension outermost)
//
// The two tiles take turns: while the threads of one are at their exponentials, the
// tensor core has the other's products, each about 1,024 cycles of either. O stays
// in TMEM; it is scaled when a row's maximum has grown by more than 2^8 over the
// one in use (the quotient by the sum undoes any common factor, and f32 has room),
// so after the first positions hardly ever.
//
// Roles (320 threads, one CTA per SM: all 512 TMEM columns): warps 0-3 and 4-7 the
// rows of tile 0 and 1, warp 8 the copies (TMA, keys and values in turn through a
// ring of four 32 KB stages), warp 9 the MMAs. P is rounded to the element type as
// in attn_shared.cu. Every wait is bounded; one that gives up sets an error word
// (bit 128 of loom_cuda_device_error), leaves NaN in the CTA's rows and ends.
#include <cuda.h>  // CUtensorMap (the encoder is reached through the runtime's driver entry point)

#include <type_traits>

#include "attn_shared.cuh"
#include "umma.cuh"

namespace loom {
namespace {

constexpr int AP_THREADS = 320, AP_N = 128, AP_STAGES = 4;
constexpr size_t AP_BLOCK = 128 * 128;           // 128 rows of 64 elements, swizzled in 128-byte rows
constexpr uint32_t AP_POLLS = 1u << 20;
constexpr float AP_LAZY = 8.0f;                  // log2 of the growth that scales O

struct ApBars {
    uint64_t full[AP_STAGES], empty[AP_STAGES], s_full[2], p_full[2], o_full[2];
    uint64_t drain;
    uint32_t tmem;
    int err, issued;  // a wait gave up; copies issued
};

__device__ int g_ap_err;  // a wait of any launch gave up

template <int NB> constexpr size_t ap_smem() {  // queries of two tiles, the ring, barriers, alignment
    return (2 + AP_STAGES) * NB * AP_BLOCK + sizeof(ApBars) + 1024;
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
__device__ __forceinline__ void ap_tma(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
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
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void ap_arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// NB: blocks of 64 dimensions (head_dim <= 64 NB)
template <class T, int NB>
__global__ void __launch_bounds__(AP_THREADS, 1)
    k_attn_prefix(AttnArgs a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv) {
    extern __shared__ uint8_t ap_raw[];
    pdl_trigger_();
    const uint32_t sm0 = (smem_u32(ap_raw) + 1023) & ~1023u;
    uint8_t *smp = ap_raw + (sm0 - smem_u32(ap_raw));
    const uint32_t ring = sm0 + 2 * NB * AP_BLOCK;
    ApBars &B = *reinterpret_cast<ApBars *>(smp + (2 + AP_STAGES) * NB * AP_BLOCK);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, hd = a.hd;
    const Item<T> it = item_of<T>(a, blockIdx.x, kvh);
    const int n = (it.p1 - it.p0 + AP_N - 1) / AP_N, rows = it.r1 - it.r0, tiles = rows > 128 ? 2 : 1;
    volatile int *err = &B.err;
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        if (*err) return false;
        if (mbar_wait_hint(bar, parity, AP_POLLS, 2000)) return true;
        *err = 1;
        return false;
    };
    auto fetch = [&](int i) {  // item i of the ring: keys (even) or values of 128 positions
        const int s = i % AP_STAGES;
        mbar_expect_tx(&B.full[s], (uint32_t)(NB * AP_BLOCK));
        B.issued = i + 1;
        for (int b = 0; b < NB; b++)
            ap_tma(ring + (uint32_t)((s * NB + b) * AP_BLOCK), i & 1 ? &mv : &mk, b * 64, it.p0 + (i >> 1) * AP_N, kvh, &B.full[s]);
    };
    if (warp == 8 && lane == 0) {
        for (int s = 0; s < AP_STAGES; s++) {
            mbar_init_nf(&B.full[s], 1);
            mbar_init_nf(&B.empty[s], 1);
        }
        for (int t = 0; t < 2; t++) {
            mbar_init_nf(&B.s_full[t], 1);
            mbar_init_nf(&B.p_full[t], 128);
            mbar_init_nf(&B.o_full[t], 1);
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
        *reinterpret_cast<uint4 *>(smp + (size_t)(tl * NB + c / 8) * AP_BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
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
        if (lane == 0) {
            const uint32_t id_s = ap_idesc<T>(AP_N, false), id_o = ap_idesc<T>((hd + 15) / 16 * 16, true);
            const int ks = (hd + 15) / 16;
            auto qk = [&](int t, int j) {  // S_t = Q_t K(j)^T
                const uint32_t q = sm0 + (uint32_t)(t * NB * AP_BLOCK), k = ring + (uint32_t)((2 * j % AP_STAGES) * NB * AP_BLOCK);
                for (int s = 0; s < ks; s++) {
                    const uint32_t off = (uint32_t)((s >> 2) * AP_BLOCK + (s & 3) * 32);
                    ap_mma_ss(tmem + t * 128, ap_desc_k(q + off), ap_desc_k(k + off), id_s, s > 0);
                }
                umma_commit(&B.s_full[t]);
            };
            auto item = [&](int i) { return wait(&B.full[i % AP_STAGES], (i / AP_STAGES) & 1); };
            bool ok = item(0);
            tc_fence_after();
            for (int t = 0; t < tiles && ok; t++) qk(t, 0);
            if (ok) umma_commit(&B.empty[0]);
            for (int j = 0; j < n && ok; j++) {
                ok = item(2 * j + 1) && (j + 1 >= n || item(2 * j + 2));
                const uint32_t v = ring + (uint32_t)(((2 * j + 1) % AP_STAGES) * NB * AP_BLOCK);
                for (int t = 0; t < tiles && ok; t++) {
                    ok = wait(&B.p_full[t], j & 1);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int s = 0; s < AP_N / 16; s++)
                        ap_mma_ts(tmem + 256 + t * 128, tmem + t * 128 + s * 8, ap_desc_mn(v + s * 2048), id_o, j > 0 || s > 0);
                    if (t == tiles - 1) umma_commit(&B.empty[(2 * j + 1) % AP_STAGES]);
                    if (j + 1 < n)
                        qk(t, j + 1);
                    else
                        umma_commit(&B.o_full[t]);
                }
                if (ok && j + 1 < n) umma_commit(&B.empty[(2 * j + 2) % AP_STAGES]);
            }
        }
        __syncwarp();
    } else if (warp / 4 < tiles) {
        const int t = warp / 4, row = it.r0 + t * 128 + (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), ts = lanes + t * 128, to = lanes + 256 + t * 128;
        float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        bool ok = true;
        for (int j = 0; j < n && ok; j++) {
            ok = wait(&B.s_full[t], j & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            uint32_t s[128];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(ts + c * 32, s + c * 32);
            tmem_wait_ld();
            const int left = it.p1 - (it.p0 + j * AP_N);
            if (left < AP_N)
#pragma unroll
                for (int c = 0; c < 128; c++)
                    if (c >= left) s[c] = 0xFF800000u;  // -inf
            float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int c = 0; c < 128; c += 4)
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = fmaxf(x[k], __uint_as_float(s[c + k]));
            const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * a.scale;  // scale >= 0
            if (__any_sync(0xffffffffu, top > m + AP_LAZY || (m == -INFINITY && top > m))) {
                const float mn = fmaxf(m, top), f = m == -INFINITY ? 0.0f : ex2(m - mn);
                l0 *= f;
                l1 *= f;
                m = mn;
                if (j) {
#pragma unroll 1
                    for (int c = 0; c < NB * 64; c += 16) {
                        uint32_t o[16];
                        tmem_ld16(to + c, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int k = 0; k < 16; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                        tmem_st16(to + c, o);
                    }
                }
            }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int h = 0; h < 4; h++) {
                uint32_t p[16];
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    const float e0 = ex2(fmaf(__uint_as_float(s[h * 32 + 2 * c]), a.scale, -base));
                    const float e1 = ex2(fmaf(__uint_as_float(s[h * 32 + 2 * c + 1]), a.scale, -base));
                    l0 += e0;
                    l1 += e1;
                    p[c] = pack2<T>(e0, e1);
                }
                tmem_st16(ts + h * 16, p);
            }
            tmem_wait_st();
            tc_fence_before();
            ap_arrive(&B.p_full[t]);
        }
        if (ok) ok = __all_sync(0xffffffffu, wait(&B.o_full[t], 0));
        if (ok) {
            tc_fence_after();
            const bool in = row < it.r1;
            const size_t at = in ? part_at(a, it.slot, row, kvh) : 0;
            if (in) a.ml[at] = make_float2(m, l0 + l1);
            float *dst = a.acc + at * hd;
            for (int c = 0; c < hd; c += 32) {
                uint32_t o[32];
                tmem_ld32(to + c, o);
                tmem_wait_ld();
                if (in)
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        if (c + k < hd)  // hd is a multiple of 8
                            *reinterpret_cast<uint4 *>(dst + c + k) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (*err) {  // what was issued ends before the memory it uses is given back
        if (warp == 9 && lane == 0) {
            umma_commit(&B.drain);
            mbar_wait_hint(&B.drain, 0, 1u << 12, 2000);
            for (int i = max(B.issued - AP_STAGES, 0); i < B.issued; i++)
                mbar_wait_hint(&B.full[i % AP_STAGES], (i / AP_STAGES) & 1, 1u << 12, 2000);
            atomicOr(&g_ap_err, 128);
        }
        for (int j = tid; j < rows; j += AP_THREADS) a.ml[part_at(a, it.slot, it.r0 + j, kvh)] = make_float2(NAN, NAN);
        __syncthreads();
    }
    tc_fence_after();
    if (warp == 9) tmem_free(tmem, 512);
}

typedef CUresult (*ApEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
ApEncodeFn ap_encoder() {
    static ApEncodeFn f = nullptr;
    if (!f) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            f = reinterpret_cast<ApEncodeFn>(p);
    }
    return f;
}

// [KV heads][positions][head_dim] of a cache in boxes of 128 positions x 64
// dimensions; what lies outside reads as zero
template <class T> bool ap_map(CUtensorMap &m, const AttnArgs &a, const void *base) {
    ApEncodeFn enc = ap_encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)a.hd, (cuuint64_t)a.prefix, (cuuint64_t)a.nkv};
    const cuuint64_t strides[2] = {(cuuint64_t)a.ppos * 2, (cuuint64_t)(a.nkv > 1 ? a.phead : a.ppos) * 2};
    const cuuint32_t box[3] = {64, AP_N, 1}, es[3] = {1, 1, 1};
    return enc(&m, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
               const_cast<void *>(base), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int NB> cudaError_t ap_launch(const AttnArgs &a, const CUtensorMap &mk, const CUtensorMap &mv, cudaStream_t st) {
    if (const cudaError_t e = allow_smem<k_attn_prefix<T, NB>>(ap_smem<NB>()); e != cudaSuccess) return e;
    k_attn_prefix<T, NB><<<dim3(a.n_pre * a.pre_tiles, a.nkv), AP_THREADS, ap_smem<NB>(), st>>>(a, mk, mv);
    count_launch();
    return cudaGetLastError();
}

template <class T> bool ap_run(const AttnArgs &a, cudaStream_t st, cudaError_t *e) {
    CUtensorMap mk, mv;
    if (!ap_map<T>(mk, a, a.pk) || !ap_map<T>(mv, a, a.pv)) return false;
    *e = a.hd <= 64 ? ap_launch<T, 1>(a, mk, mv, st) : ap_launch<T, 2>(a, mk, mv, st);
    return true;
}

}  // namespace

int attn_prefix_error() {
    int v = 0;
    return cudaMemcpyFromSymbol(&v, g_ap_err, sizeof v) == cudaSuccess ? v : -1;
}

bool attn_prefix_run(int type, const AttnArgs &a, cudaStream_t st, cudaError_t *e) {
    return type == T_F16 ? ap_run<__half>(a, st, e) : ap_run<__nv_bfloat16>(a, st, e);
}

}  // namespace loom
