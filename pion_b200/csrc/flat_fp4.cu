// Products of a query batch with microscaled 4-bit rows, and the k best rows of each query,
// on B200 (sm_100a).  No counterpart in the reference.
//
//   score(t, r) = f32(((sum_j q[t][j] v[r][j]) g_r) g_t),  q and v in units of their row's g
//
// Kernels:
//   fp4_tc_kernel     the product on tcgen05 (kind::mxf4 / mxf4nvf4 with block scales).  Index
//                     rows are the UMMA M side, streamed by TMA; a tile of queries is the N
//                     side and stays in shared memory.  TMEM lane = row, so one query's
//                     scores leave the warp in row order, 128 bytes at a time, and one query
//                     costs a 16-column MMA beside the stream.  Epilogues: write the scores,
//                     or keep the rows that reach a query's threshold.
//   theta_kernel      a query's threshold from its scores of a sample of the rows.
//   finish_kernel     the k best of a query: its candidates scored exactly, sorted.
//
// Exactness: a product of two codes is a multiple of 1/4 up to 36, and a row's scales span a
// few powers of two, so the sum in float64 is exact; it is rounded once to float32, and rows
// with equal scores rank by id.  The tensor cores' float32 sums only choose which rows are
// summed again: with |approximate - exact| <= eps, a row among the k best scores at least
// the k-th best approximate score of any subset less 2 eps.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "fp4.cuh"
#include "internal.h"

namespace pion {
namespace fp4 {

constexpr int ROWS = 128;                // rows per CTA tile (UMMA M per CTA, TMEM lanes)
constexpr int KC = 128;                  // code bytes of K per pipeline stage (256 elements)
constexpr int A_BYTES = ROWS * KC;       // 16 KB
constexpr int EPI_WARPS = 8;             // two per TMEM lane quarter, alternate column chunks
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t TMEM_COLS = 512;
constexpr int MAX_STAGES = 8;
constexpr int SMEM_MAX = 232448;         // 227 KB
constexpr int CAP = 4096;                // candidates kept per query
constexpr int LIST = 2048;               // of which at most this many are scored exactly

// 512-byte scale atoms per stage of 256 elements
__host__ __device__ constexpr int atoms_per_stage(int fmt) { return fmt == kMX ? 2 : 4; }

// Error bound of an approximate score: eps = rel_eps(dp) * |q| * |v| (norms bounded from the
// block scales): two float32 steps of the running sum for every 64 elements, and eight more.
// Measured over blocks of many magnitudes and q near v, where partial sums are largest:
// 2^-23.5 at 64 elements, 2^-21.0 at 1536 and 2^-18.8 at 8192 (the bound: 2^-18.8, 2^-17.0
// and 2^-14.9).
__host__ __device__ constexpr float rel_eps(int dp) { return (float)(dp / 64 + 8) * 0x1p-22f; }

enum Mode { kScores = 0, kCollect = 1 };

struct TcParams {
    const float* row_scale;   // [n_rows]
    const float* q_scale;     // [query slot]
    int64_t n_rows;
    int nq;
    int nt, nt_pad;           // queries per tile, and their slots (a multiple of 128)
    int n_qt;
    int kchunks;              // stages per tile
    int mmas;                 // 64-element steps per tile
    int atoms;                // scale atoms per row tile
    int stages;
    int n_tiles;              // row tiles of this launch ...
    int tile_step;            // ... the j-th being tile j * tile_step
    // kScores
    void* out;                // [nq][ld]; column = position of the row in this launch
    int out_type;
    int64_t ld;
    // kCollect
    const float* theta;       // [nq]: least score / q_scale kept
    int* cand_n;              // [nq]
    uint64_t* cand;           // [nq][CAP]: approximate score bits << 32 | row
    int* status;
    uint64_t wait_ns;
};

// Shared-memory plan of one launch.
struct Plan {
    int nt, nt_pad, n_qt, kchunks, stages;
    int b_bytes, sfb_bytes, stage_bytes, smem;
};

// ------------------------------------------------------------- PTX pieces --
// Scale atoms in shared memory: 32 rows of 16 bytes, no swizzle, 8-row groups 128 B apart.
__device__ __forceinline__ uint64_t make_scale_desc(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>(128u >> 4) << 16;
    d |= static_cast<uint64_t>(128u >> 4) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    return d;
}

// Instruction descriptor of the block-scaled kinds: e2m1 x e2m1 -> f32, both K-major.
template <int FMT>
__host__ __device__ constexpr uint32_t make_idesc_fp4(int m, int n) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           ((FMT == kMX ? 1u : 0u) << 23) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void tc_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
}

template <int FMT>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
    if (FMT == kMX)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X"
            " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X"
            " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// Orders floats as unsigned integers; NaN is put below everything by the callers.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}

template <class T>
__device__ __forceinline__ T cast_out(float v);
template <>
__device__ __forceinline__ float cast_out<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 cast_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half cast_out<__half>(float v) { return __float2half_rn(v); }

// One 32-column chunk of one row's scores to out[t][col], t from t0.
template <class T>
__device__ __forceinline__ void store_chunk(const uint32_t (&r)[32], const TcParams& p, int t0,
                                            int n, int64_t col, const float* gq, float g) {
    T* out = static_cast<T*>(p.out) + (int64_t)t0 * p.ld + col;
    const bool row_ok = g == g;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        if (j < n) {
            const float s = gq[j];
            const float v = row_ok && s == s ? __uint_as_float(r[j]) * g * s : -INFINITY;
            out[(int64_t)j * p.ld] = cast_out<T>(v);
        }
    }
}

// ------------------------------------------------------------ the product --
// Warp 0 loads, warp 1 issues the MMAs, the others drain TMEM.  Accumulators are double
// buffered at columns 0 and nt; above them two sets of scale columns, used in turn.  A set is
// written again only after the MMAs that read it are done (sfree).
template <int FMT>
__global__ void __launch_bounds__(THREADS, 1)
    fp4_tc_kernel(const __grid_constant__ CUtensorMap tmap_rows,
                  const __grid_constant__ CUtensorMap tmap_row_sf,
                  const __grid_constant__ CUtensorMap tmap_q,
                  const __grid_constant__ CUtensorMap tmap_q_sf, TcParams p, int mode) {
    constexpr int APS = atoms_per_stage(FMT);
    constexpr int STAGE = A_BYTES + APS * 512;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const int nt = p.nt;
    const int sf_tiles = p.nt_pad / 128;
    uint8_t* ring = smem;                                    // stages x (codes, scale atoms)
    uint8_t* sB = ring + p.stages * STAGE;                   // [kchunk][query][128 B], swizzled
    uint8_t* sSF = sB + p.kchunks * nt * KC;                 // [128-query tile][kchunk][APS]
    float* s_gq = reinterpret_cast<float*>(sSF + sf_tiles * p.kchunks * APS * 512);
    float* s_th = s_gq + 256;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_th + 256);
    uint64_t* empty = full + MAX_STAGES;
    uint64_t* tfull = empty + MAX_STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* sfree = tempty + 2;
    uint64_t* bfull = sfree + 2;
    uint64_t* drain = bfull + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int qt = blockIdx.x % p.n_qt;
    const int lanes_of_work = gridDim.x / p.n_qt;  // CTAs per query tile
    const int first = blockIdx.x / p.n_qt;

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], EPI_WARPS);
            mbar_init(&sfree[b], 1);
        }
        mbar_init(bfull, 1);
        mbar_init(drain, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    for (int j = threadIdx.x; j < 256; j += THREADS) {
        const int t = qt * nt + j;
        const bool ok = j < nt && t < p.nq;
        s_gq[j] = ok ? p.q_scale[(int64_t)qt * p.nt_pad + j] : 0.0f;
        s_th[j] = ok && mode == kCollect ? p.theta[t] : INFINITY;
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        if (lane == 0) {
            tma_prefetch_desc(&tmap_rows);
            tma_prefetch_desc(&tmap_row_sf);
            mbar_arrive_expect_tx(bfull, (uint32_t)(p.kchunks * nt * KC +
                                                    sf_tiles * p.kchunks * APS * 512));
            for (int kc = 0; kc < p.kchunks; ++kc) {
                tma_load_2d(sB + kc * nt * KC, &tmap_q, bfull, kc * KC, qt * p.nt_pad);
                for (int h = 0; h < sf_tiles; ++h)
                    tma_load_2d(sSF + (h * p.kchunks + kc) * APS * 512, &tmap_q_sf, bfull, 0,
                                (qt * sf_tiles + h) * p.atoms + kc * APS);
            }
            int stage = 0;
            uint32_t phase = 0, issued = 0, parity = 0;  // bits by stage
            bool ok = true;
            for (int j = first; j < p.n_tiles && ok; j += lanes_of_work) {
                const int tile = j * p.tile_step;
                for (int kc = 0; kc < p.kchunks; ++kc) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, p.status, abort_flag, p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = ring + stage * STAGE;
                    mbar_arrive_expect_tx(&full[stage], STAGE);
                    tma_load_2d(dst, &tmap_rows, &full[stage], kc * KC, tile * ROWS);
                    tma_load_2d(dst + A_BYTES, &tmap_row_sf, &full[stage], 0,
                                tile * p.atoms + kc * APS);
                    issued |= 1u << stage;
                    parity = (parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every copy this thread issued lands before the CTA may exit.
            mbar_wait(bfull, 0, p.status, nullptr, p.wait_ns);
            for (int s = 0; s < p.stages; ++s)
                if ((issued >> s) & 1u)
                    mbar_wait(&full[s], (parity >> s) & 1u, p.status, nullptr, p.wait_ns);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------- MMA issuer
        if (lane == 0) {
            const uint32_t idesc = make_idesc_fp4<FMT>(ROWS, nt);
            const uint32_t sf_set = APS * 4 * (1 + sf_tiles);
            const uint32_t sf_base = tmem_base + 2 * nt;
            int stage = 0;
            uint32_t phase = 0;
            uint32_t it = 0;
            bool ok = mbar_wait(bfull, 0, p.status, abort_flag, p.wait_ns);
            int n = 0;
            for (int j = first; j < p.n_tiles && ok; j += lanes_of_work, ++n) {
                const int buf = n & 1;
                if (!mbar_wait(&tempty[buf], ((n >> 1) & 1) ^ 1, p.status, abort_flag, p.wait_ns))
                    break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * nt);
                for (int kc = 0; kc < p.kchunks; ++kc, ++it) {
                    const uint32_t set = it & 1u;
                    if (!mbar_wait(&full[stage], phase, p.status, abort_flag, p.wait_ns) ||
                        !mbar_wait(&sfree[set], ((it >> 1) & 1u) ^ 1u, p.status, abort_flag,
                                   p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a0 = smem_u32(ring + stage * STAGE);
                    const uint32_t b0 = smem_u32(sB + kc * nt * KC);
                    const uint32_t sfa = sf_base + set * sf_set, sfb = sfa + APS * 4;
#pragma unroll
                    for (int a = 0; a < APS; ++a) {
                        tc_cp_scales(sfa + a * 4, make_scale_desc(a0 + A_BYTES + a * 512));
                        for (int h = 0; h < sf_tiles; ++h)
                            tc_cp_scales(sfb + (a * sf_tiles + h) * 4,
                                         make_scale_desc(smem_u32(
                                             sSF + ((h * p.kchunks + kc) * APS + a) * 512)));
                    }
                    const int steps = min(4, p.mmas - kc * 4);
                    for (int kk = 0; kk < steps; ++kk) {
                        // MX: an atom's bytes 0-1 scale one 64-element step, 2-3 the next
                        const int a = FMT == kMX ? kk >> 1 : kk;
                        const uint32_t id = FMT == kMX ? (uint32_t)(kk & 1) * 2u : 0u;
                        mma_fp4<FMT>(d_tmem, make_sw128_kmajor_desc(a0 + kk * 32),
                                     make_sw128_kmajor_desc(b0 + kk * 32),
                                     idesc | (id << 4) | (id << 29), sfa + a * 4,
                                     sfb + a * sf_tiles * 4, (kc | kk) != 0 ? 1u : 0u);
                    }
                    tc_commit(&empty[stage]);
                    tc_commit(&sfree[set]);
                    if (++stage == p.stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                tc_commit(&tfull[buf]);
            }
            // All MMAs issued above complete before TMEM is released.
            tc_commit(drain);
            mbar_wait(drain, 0, p.status, nullptr, p.wait_ns);
        }
    } else {
        // ---------------------------------------------------------- epilogue
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2;
        const int chunks = (nt + 31) / 32;
        int n = 0;
        for (int j = first; j < p.n_tiles; j += lanes_of_work, ++n) {
            const int buf = n & 1;
            const int in_tile = quarter * 32 + lane;
            const int64_t row = (int64_t)j * p.tile_step * ROWS + in_tile;
            const bool row_in = row < p.n_rows;
            const float g = row_in ? __ldg(&p.row_scale[row]) : __int_as_float(0x7fc00000);
            const bool got = mbar_wait(&tfull[buf], (n >> 1) & 1, p.status, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, got)) break;
            tc_fence_after();
            const uint32_t taddr =
                tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * nt);
            for (int c = half; c < chunks; c += 2) {
                uint32_t r[32];
                __syncwarp();
                tmem_ld32(taddr + c * 32, r);
                tmem_ld_wait_regs(r);
                const int t0 = qt * nt + c * 32;
                const int cols = min(32, min(nt - c * 32, p.nq - t0));
                if (mode == kScores) {
                    if (row_in && cols > 0) {
                        const int64_t col = (int64_t)j * ROWS + in_tile;
                        if (p.out_type == PION_B200_F32)
                            store_chunk<float>(r, p, t0, cols, col, s_gq + c * 32, g);
                        else if (p.out_type == PION_B200_BF16)
                            store_chunk<__nv_bfloat16>(r, p, t0, cols, col, s_gq + c * 32, g);
                        else
                            store_chunk<__half>(r, p, t0, cols, col, s_gq + c * 32, g);
                    }
                } else {
                    const float* th = s_th + c * 32;
                    bool any = false;
#pragma unroll
                    for (int i = 0; i < 32; ++i) any |= __uint_as_float(r[i]) * g >= th[i];
                    if (any) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float v = __uint_as_float(r[i]) * g;
                            if (v >= th[i]) {
                                const int t = t0 + i;
                                const int at = atomicAdd(&p.cand_n[t], 1);
                                if (at < CAP)
                                    p.cand[(int64_t)t * CAP + at] =
                                        ((uint64_t)__float_as_uint(v * s_gq[c * 32 + i]) << 32) |
                                        (uint32_t)row;
                            }
                        }
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[buf]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// --------------------------------------------------------------- selection --
constexpr int SEL = 256;  // threads of a selection CTA

// The k-th largest (1-based) of m ordered values, by the CTA: four passes over byte
// histograms.  `value(i)` is called once per pass for every i.
template <class F>
__device__ uint32_t kth_largest(int m, int k, int* hist, F value) {
    __shared__ uint32_t s_prefix;
    __shared__ int s_left;
    uint32_t prefix = 0;
    int left = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int b = threadIdx.x; b < 256; b += SEL) hist[b] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < m; i += SEL) {
            const uint32_t o = value(i);
            if (shift == 24 || (o >> (shift + 8)) == (prefix >> (shift + 8)))
                atomicAdd(&hist[(o >> shift) & 255u], 1);
        }
        __syncthreads();
        if (threadIdx.x < 32) {
            // warp 0: lane L owns the eight bins 255 - 8 L and below
            const int lane = threadIdx.x;
            int c[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                c[j] = hist[255 - 8 * lane - j];
                sum += c[j];
            }
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += up;
            }
            before -= sum;
            if (before < left && before + sum >= left) {
                int b = before;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (b < left && b + c[j] >= left) {
                        s_prefix = prefix | ((uint32_t)(255 - 8 * lane - j) << shift);
                        s_left = left - b;
                    }
                    b += c[j];
                }
            }
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
        __syncthreads();
    }
    return prefix;
}

__device__ __forceinline__ uint32_t ordered_score(float v) { return v == v ? ordered(v) : 0u; }

// Infinite where a float32 sum could overflow: nothing is known of an approximate score then.
// The last term covers products below the least normal float.
__device__ __forceinline__ float eps_of(int dp, float q_norm, float norm_max) {
    const float size = q_norm * norm_max;
    return size < 0x1p120f ? rel_eps(dp) * size + 0x1p-100f : INFINITY;
}

// Threshold of one query per CTA: the k-th best of its approximate scores so far (the sample's,
// or the candidates of a part of the rows) less 2 eps, in units of the query's g.  Resets the
// query's candidate count.
__global__ void __launch_bounds__(SEL)
    theta_kernel(const float* sample, int64_t ld, int m, const uint64_t* cand, int k,
                 int dp, const float* q_scale, int nt, int nt_pad, const float* q_norm,
                 const float* norm_max, float* theta, int* cand_n) {
    __shared__ int hist[256];
    const int t = blockIdx.x;
    const float* s = sample + (int64_t)t * ld;
    const uint64_t* c = cand + (int64_t)t * CAP;
    if (cand) m = min(cand_n[t], CAP);
    const float gq = q_scale[query_slot(t, nt, nt_pad)];
    float th = INFINITY;  // an empty or zero query collects nothing
    if (gq > 0.0f) {
        th = -INFINITY;
        if (cand && m < k) th = theta[t];
        if (m >= k) {
            const uint32_t o = kth_largest(m, k, hist, [&](int i) {
                return ordered_score(cand ? __uint_as_float((uint32_t)(c[i] >> 32)) : s[i]);
            });
            const float kth = o ? unordered(o) : -INFINITY;
            const float low = kth - 2.0f * eps_of(dp, q_norm[t], *norm_max);
            th = low / gq;
            th = th > -INFINITY ? th - 0x1p-20f * fabsf(th) : -INFINITY;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        theta[t] = th;
        cand_n[t] = 0;
    }
}

struct FinishParams {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scale;
    const float* norm_max;
    int64_t n_rows;
    int64_t id_base;
    int dp, atoms;
    const uint8_t* q_codes;
    const uint8_t* q_scales;
    const float* q_scale;
    const float* q_norm;
    int nt, nt_pad;
    int k;
    const float* dense;      // [nq][ld] scores of every row, or null
    int64_t ld;
    const int* cand_n;       // else the candidates
    const uint64_t* cand;
    int32_t* out_ids;        // [nq][k]
    float* out_scores;
};

// Query block scales as float, codes as bytes (twice their value).
struct QueryShared {
    int8_t* codes;
    float* scales;
};

// sum_j q_j v_j in units of both g, by one warp: exact integer sums per block, float64 over
// the blocks.
template <int FMT>
__device__ __forceinline__ double warp_dot(const FinishParams& p, const QueryShared& q,
                                           int64_t row, int lane) {
    const uint4* codes = reinterpret_cast<const uint4*>(p.codes + row * (p.dp / 2));
    double acc = 0.0;
    for (int b = lane; b < p.dp / 32; b += 32) {  // 32 elements per lane
        const uint4 w = __ldg(codes + b);
        const uint32_t raw[4] = {w.x, w.y, w.z, w.w};
        const int4* qb = reinterpret_cast<const int4*>(q.codes + b * 32);
        int dot[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int4 qq = qb[h];
            dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h]), qq.x, dot[h]);
            dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h] >> 16), qq.y, dot[h]);
            dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h + 1]), qq.z, dot[h]);
            dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h + 1] >> 16), qq.w, dot[h]);
        }
        if (FMT == kMX) {
            const float s =
                e8m0_value(__ldg(p.scales + scale_word(row, b >> 2, p.atoms) + (b & 3)));
            acc += (double)(dot[0] + dot[1]) * ((double)q.scales[b] * (double)s);
        } else {
            const uint8_t* at = p.scales + scale_word(row, b >> 1, p.atoms) + (b & 1) * 2;
            const uint32_t two = __ldg(reinterpret_cast<const uint16_t*>(at));
            acc += (double)dot[0] * ((double)q.scales[2 * b] * (double)e4m3_value(two & 255u));
            acc += (double)dot[1] * ((double)q.scales[2 * b + 1] * (double)e4m3_value(two >> 8));
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    return 0.25 * acc;
}

// Larger is better: (score desc, row asc); 0 for a row that cannot be found.
__device__ __forceinline__ uint64_t row_key(double dot, float g, float gq, int64_t row) {
    const float s = (float)((dot * (double)g) * (double)gq) + 0.0f;
    if (!(s > -INFINITY)) return 0;
    return ((uint64_t)ordered(s) << 32) | (uint32_t)~(uint32_t)row;
}

// Sorts n <= LIST keys in shared memory, largest first (bitonic over the next power of two;
// the rest is filled with zeros).
__device__ void sort_desc(uint64_t* key, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += SEL) key[i] = 0;
    __syncthreads();
    for (int w = 2; w <= size; w <<= 1)
        for (int s = w >> 1; s; s >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += SEL) {
                const int a = 2 * i - (i & (s - 1));
                const int b = a + s;
                const bool desc = (a & w) == 0;
                const uint64_t x = key[a], y = key[b];
                if ((x < y) == desc) {
                    key[a] = y;
                    key[b] = x;
                }
            }
            __syncthreads();
        }
}

// The k best rows of one query per CTA.
template <int FMT>
__global__ void __launch_bounds__(SEL) finish_kernel(FinishParams p) {
    __shared__ __align__(16) uint64_t key[LIST];
    __shared__ int hist[256];
    __shared__ int s_n;
    extern __shared__ __align__(16) uint8_t dyn[];  // query bytes [dp], scales [dp / block]
    const int t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int W = SEL / 32;
    const int64_t qs = query_slot(t, p.nt, p.nt_pad);
    const float gq = p.q_scale[qs];
    QueryShared q;
    q.codes = reinterpret_cast<int8_t*>(dyn);
    q.scales = reinterpret_cast<float*>(dyn + p.dp);

    int found = 0;
    if (gq > 0.0f) {
        for (int i = threadIdx.x; i < p.dp / 4; i += SEL)
            reinterpret_cast<uint32_t*>(q.codes)[i] = e2m1x4_bytes(
                reinterpret_cast<const uint16_t*>(p.q_codes + qs * (p.dp / 2))[i]);
        for (int b = threadIdx.x; b < p.dp / block_of(FMT); b += SEL)
            q.scales[b] = scale_value<FMT>(p.q_scales[scale_word(qs, b >> 2, p.atoms) + (b & 3)]);
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        const float two_eps = 2.0f * eps_of(p.dp, p.q_norm[t], *p.norm_max);
        const float* dense = p.dense ? p.dense + (int64_t)t * p.ld : nullptr;
        const uint64_t* cand = p.dense ? nullptr : p.cand + (int64_t)t * CAP;
        const int m = p.dense ? (int)p.n_rows : p.cand_n[t];
        const bool known = two_eps < INFINITY;  // else any row may be among the best
        bool whole = !p.dense && (m > CAP || !known);
        if (!whole) {
            auto approx = [&](int i) {
                return dense ? dense[i] : __uint_as_float((uint32_t)(cand[i] >> 32));
            };
            float cut = -INFINITY;
            if (m > p.k) {
                const uint32_t o =
                    kth_largest(m, p.k, hist, [&](int i) { return ordered_score(approx(i)); });
                cut = o ? unordered(o) - two_eps : -INFINITY;
            }
            for (int i = threadIdx.x; i < m; i += SEL) {
                const float a = approx(i);
                if (a >= cut || !known) {
                    const int at = atomicAdd(&s_n, 1);
                    if (at < LIST) key[at] = dense ? (uint64_t)i : (cand[i] & 0xFFFFFFFFu);
                }
            }
            __syncthreads();
            whole = s_n > LIST;
            if (!whole) {
                for (int i = warp; i < s_n; i += W) {
                    const int64_t row = (int64_t)key[i];
                    const double dot = warp_dot<FMT>(p, q, row, lane);
                    if (lane == 0) key[i] = row_key(dot, p.row_scale[row], gq, row);
                }
                __syncthreads();
                found = s_n;
                sort_desc(key, found);
            }
        }
        if (whole) {
            // More rows than fit reach the threshold (many equal rows, a sample that missed
            // the best ones, or norms past float32): every row exactly, keeping the rows that
            // beat the k-th best so far.
            if (threadIdx.x == 0) s_n = 0;
            __syncthreads();
            uint64_t floor_key = 0;
            constexpr int BATCH = 512;
            for (int64_t r0 = 0; r0 < p.n_rows; r0 += BATCH) {
                for (int i = warp; i < BATCH; i += W) {
                    const int64_t row = r0 + i;
                    if (row >= p.n_rows) break;
                    const float g = __ldg(&p.row_scale[row]);
                    if (!(g == g)) continue;
                    const double dot = warp_dot<FMT>(p, q, row, lane);
                    const uint64_t x = row_key(dot, g, gq, row);
                    if (lane == 0 && x > floor_key) key[atomicAdd(&s_n, 1)] = x;
                }
                __syncthreads();
                const int have = s_n;
                if (have > LIST - BATCH || r0 + BATCH >= p.n_rows) {
                    sort_desc(key, have);
                    found = min(have, p.k);
                    floor_key = found == p.k ? key[p.k - 1] : 0;
                    __syncthreads();
                    if (threadIdx.x == 0) s_n = found;
                }
                __syncthreads();
            }
        }
    } else if (gq == 0.0f) {
        // Every row that holds anything scores 0: the first k of them.
        if (threadIdx.x == 0) s_n = 0;
        __syncthreads();
        for (int64_t r0 = 0; r0 < p.n_rows && found < p.k; r0 += SEL) {
            const int64_t row = r0 + threadIdx.x;
            const float g = row < p.n_rows ? p.row_scale[row] : __int_as_float(0x7fc00000);
            const unsigned live = __ballot_sync(0xffffffffu, g == g);
            if (lane == 0) hist[warp] = __popc(live);
            __syncthreads();
            int at = found;
            int all = 0;
            for (int w = 0; w < W; ++w) {
                if (w < warp) at += hist[w];
                all += hist[w];
            }
            at += __popc(live & ((1u << lane) - 1u));
            if (g == g && at < p.k) key[at] = ((uint64_t)ordered(0.0f) << 32) | (uint32_t)~(uint32_t)row;
            found += all;
            __syncthreads();
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < p.k; j += SEL) {
        const uint64_t x = j < found ? key[j] : 0;
        p.out_ids[(int64_t)t * p.k + j] =
            x ? (int32_t)(p.id_base + (int64_t)(uint32_t)~(uint32_t)x) : -1;
        p.out_scores[(int64_t)t * p.k + j] = x ? unordered((uint32_t)(x >> 32)) : -INFINITY;
    }
}

static int round_up(int x, int a) { return (x + a - 1) / a * a; }

// Queries per tile: as many as the accumulators' two buffers and two sets of scale columns
// leave of the 512 TMEM columns, and shared memory beside at least three stages; spread
// evenly over the tiles.
static bool make_plan(int fmt, int dp, int nq, Plan* out) {
    const int aps = atoms_per_stage(fmt);
    Plan s;
    s.kchunks = (dp / 2 + KC - 1) / KC;
    s.stage_bytes = A_BYTES + aps * 512;
    const int fixed = 1024 + 2 * 256 * 4 + (2 * MAX_STAGES + 8) * 8 + 64;
    int most = 0;
    for (int nt = 16; nt <= 208; nt += 16) {
        const int pad = round_up(nt, 128);
        const int cols = 2 * nt + 2 * aps * 4 * (1 + pad / 128);
        const int bytes = fixed + s.kchunks * (nt * KC + pad / 128 * aps * 512) + 3 * s.stage_bytes;
        // 16 columns past an odd number of 16s are read with the last chunk
        if (cols <= (int)TMEM_COLS && bytes <= SMEM_MAX) most = nt;
    }
    if (most == 0) return false;
    s.n_qt = (nq + most - 1) / most;
    s.nt = round_up((nq + s.n_qt - 1) / s.n_qt, 16);
    s.n_qt = (nq + s.nt - 1) / s.nt;
    s.nt_pad = round_up(s.nt, 128);
    s.b_bytes = s.kchunks * s.nt * KC;
    s.sfb_bytes = s.kchunks * (s.nt_pad / 128) * aps * 512;
    s.stages = (SMEM_MAX - fixed - s.b_bytes - s.sfb_bytes) / s.stage_bytes;
    s.stages = s.stages > MAX_STAGES ? MAX_STAGES : s.stages;
    s.smem = fixed + s.b_bytes + s.sfb_bytes + s.stages * s.stage_bytes;
    *out = s;
    return true;
}

}  // namespace fp4

int fp4_max_dim() { return fp4::kMaxDim; }
int fp4_cap() { return fp4::CAP; }
int fp4_tile_rows() { return fp4::ROWS; }

bool fp4_plan(int format, int dp, int nq, Fp4Plan* out) {
    fp4::Plan s;
    if (!fp4::make_plan(format, dp, nq, &s)) return false;
    out->nt = s.nt;
    out->nt_pad = s.nt_pad;
    out->n_qt = s.n_qt;
    return true;
}

int launch_fp4_product(const Fp4Product& L, cudaStream_t st) {
    using namespace fp4;
    Plan s;
    const int dp = pad_dim(L.dim);
    if (!make_plan(L.format, dp, L.nq, &s)) return PION_B200_ESHAPE;
    const int atoms = atoms_of(L.format, dp), aps = atoms_per_stage(L.format);
    const int64_t row_tiles = (L.n_rows + ROWS - 1) / ROWS;
    const int64_t store_tiles = (L.store_rows + 127) / 128;
    CUtensorMap rows, row_sf, q, q_sf;
    if (make_tmap_2d(&rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, L.codes, (uint64_t)dp / 2,
                     (uint64_t)L.store_rows, (uint64_t)dp / 2, KC, ROWS,
                     CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
        make_tmap_2d(&row_sf, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, L.scales, 128,
                     (uint64_t)store_tiles * atoms, 512, 128, (uint32_t)aps,
                     CU_TENSOR_MAP_SWIZZLE_NONE) != 0 ||
        make_tmap_2d(&q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, L.q_codes, (uint64_t)dp / 2,
                     (uint64_t)s.n_qt * s.nt_pad, (uint64_t)dp / 2, KC, (uint32_t)s.nt,
                     CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
        make_tmap_2d(&q_sf, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, L.q_scales, 128,
                     (uint64_t)s.n_qt * (s.nt_pad / 128) * atoms, 512, 128, (uint32_t)aps,
                     CU_TENSOR_MAP_SWIZZLE_NONE) != 0)
        return PION_B200_ECUDA;
    TcParams p;
    p.row_scale = L.row_scale;
    p.q_scale = L.q_scale;
    p.n_rows = L.n_rows;
    p.nq = L.nq;
    p.nt = s.nt;
    p.nt_pad = s.nt_pad;
    p.n_qt = s.n_qt;
    p.kchunks = s.kchunks;
    p.mmas = dp / 64;
    p.atoms = atoms;
    p.stages = s.stages;
    p.n_tiles = L.n_tiles > 0 ? L.n_tiles : (int)row_tiles;
    p.tile_step = L.tile_step;
    p.out = L.out;
    p.out_type = L.out_type;
    p.ld = L.ld;
    p.theta = L.theta;
    p.cand_n = L.cand_n;
    p.cand = L.cand;
    p.status = L.status;
    p.wait_ns = L.wait_ns;
    int64_t per = L.num_sms / s.n_qt;  // CTAs per query tile: one wave where there are enough SMs
    if (per < 1) per = 1;
    if (per > p.n_tiles) per = p.n_tiles;
    const dim3 grid((unsigned)(per * s.n_qt));
    const int mode = L.theta ? kCollect : kScores;
    const bool mx = L.format == kMX;
    const void* fn = mx ? (const void*)fp4_tc_kernel<kMX> : (const void*)fp4_tc_kernel<kNV>;
    if (set_smem_limit(fn, s.smem) != 0) return PION_B200_ECUDA;
    if (mx)
        fp4_tc_kernel<kMX><<<grid, THREADS, s.smem, st>>>(rows, row_sf, q, q_sf, p, mode);
    else
        fp4_tc_kernel<kNV><<<grid, THREADS, s.smem, st>>>(rows, row_sf, q, q_sf, p, mode);
    return cudaGetLastError() == cudaSuccess ? 0 : PION_B200_ECUDA;
}

int launch_fp4_theta(const float* sample, int64_t ld, int m, const uint64_t* cand, int k, int dim,
                     const float* q_scale, int nt, int nt_pad, const float* q_norm,
                     const float* norm_max, int nq, float* theta, int* cand_n, cudaStream_t st) {
    fp4::theta_kernel<<<(unsigned)nq, fp4::SEL, 0, st>>>(sample, ld, m, cand, k,
                                                         fp4::pad_dim(dim), q_scale, nt, nt_pad,
                                                         q_norm, norm_max, theta, cand_n);
    return cudaGetLastError() == cudaSuccess ? 0 : PION_B200_ECUDA;
}

int launch_fp4_finish(const Fp4Finish& L, cudaStream_t st) {
    using namespace fp4;
    FinishParams p;
    p.codes = L.codes;
    p.scales = L.scales;
    p.row_scale = L.row_scale;
    p.norm_max = L.norm_max;
    p.n_rows = L.n_rows;
    p.id_base = L.id_base;
    p.dp = pad_dim(L.dim);
    p.atoms = atoms_of(L.format, p.dp);
    p.q_codes = L.q_codes;
    p.q_scales = L.q_scales;
    p.q_scale = L.q_scale;
    p.q_norm = L.q_norm;
    p.nt = L.nt;
    p.nt_pad = L.nt_pad;
    p.k = L.k;
    p.dense = L.dense;
    p.ld = L.ld;
    p.cand_n = L.cand_n;
    p.cand = L.cand;
    p.out_ids = L.out_ids;
    p.out_scores = L.out_scores;
    const int smem = p.dp + p.dp / block_of(L.format) * 4;
    if (L.format == kMX)
        finish_kernel<kMX><<<(unsigned)L.nq, SEL, smem, st>>>(p);
    else
        finish_kernel<kNV><<<(unsigned)L.nq, SEL, smem, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : PION_B200_ECUDA;
}

}  // namespace pion
