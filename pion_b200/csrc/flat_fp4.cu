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
//   theta_sample_kernel, theta_kernel
//                     a query's threshold from its scores of a sample of the rows, and from
//                     its candidates so far.
//   split_kernel      few queries: the candidates from the scores of every row.
//   finish_kernel     the k best of a query: its candidates scored exactly, sorted.
//   rescue_kernel     queries with more candidates than are kept: every row, exactly.
//
// Exactness: a product of two codes is a multiple of 1/4 up to 36 and a scale one of few bits, so
// sums are held as integers (or, in MX, in float64 where a row's exponents lie near enough to each
// other for that to be the same); ((sum) g_r) g_t is rounded once to float32, and rows with equal
// scores rank by id.  The tensor cores' float32 sums only choose which rows are summed again: with
// |approximate - exact| <= eps, a row among the k best scores at least the k-th best approximate
// score of any subset less 2 eps.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "fp4.cuh"
#include "internal.h"

namespace pion {
namespace fp4 {

constexpr int HALF = 128;                // rows per CTA (TMEM lanes)
constexpr int ROWS = 2 * HALF;           // rows per tile: a CTA pair (UMMA M = 256)
constexpr int KC = 128;                  // code bytes of K per pipeline stage (256 elements)
constexpr int A_BYTES = HALF * KC;       // 16 KB
// Six warpgroups: the scale warps; the loading and the MMA warp (and two idle ones); four of
// epilogue warps, four per TMEM lane quarter.  An epilogue thread holds up to 64
// accumulators, so that one buffer of them is free again as soon as it is read.
constexpr int EPI_WARPS = 16;
constexpr int PER_QUARTER = EPI_WARPS / 4;
constexpr int HELD = 8 / PER_QUARTER;    // chunks of 32 columns a warp may have of a tile
constexpr int SCALE_WARPS = 4;
constexpr int THREADS = 256 + 32 * EPI_WARPS;  // 80 registers a thread at launch ...
constexpr int REGS_SCALE = 48, REGS_ISSUE = 48, REGS_EPI = 96;  // ... and 6 * 80 in all here
static_assert(REGS_SCALE + REGS_ISSUE + (EPI_WARPS / 4) * REGS_EPI <= (THREADS / 128) * 80,
              "register split");
constexpr uint32_t TMEM_COLS = 512;
constexpr int MAX_STAGES = 8;
constexpr int MAX_NT = 256;
constexpr int SMEM_MAX = 232448;         // 227 KB
constexpr int CAP = 4096;                // candidates kept per query
constexpr int HITS = 64;                 // appended candidates an epilogue warp holds back
constexpr int LIST = 2048;               // of which at most this many are scored exactly

// 512-byte scale atoms per stage of 256 elements
__host__ __device__ constexpr int atoms_per_stage(int fmt) { return fmt == kMX ? 2 : 4; }

// Error bound of an approximate score: eps = rel_eps(dp) * |q| * |v| (norms bounded from the
// block scales): two float32 steps of the running sum for every 64 elements, and eight more.
// Measured over blocks of many magnitudes and q near v, where partial sums are largest:
// 2^-23.5 at 64 elements, 2^-21.0 at 1536 and 2^-18.8 at 8192 (the bound: 2^-18.7, 2^-17.0
// and 2^-14.9).  Where every step is cut off, one large product and all others just below its last
// bits: 2^-22.7, 2^-18.6 and 2^-16.2, about one step of the sum for every 64 elements.
__host__ __device__ constexpr float rel_eps(int dp) { return (float)(dp / 64 + 8) * 0x1p-22f; }

enum Mode { kScores = 0, kCollect = 1 };

// Shared-memory and TMEM plan of one launch.
struct Plan {
    int nt, nt_pad, n_qt;     // queries per tile, their slots (a multiple of 128), tiles
    int kchunks;              // stages per tile
    int stages;
    int bufs;                 // accumulator buffers of nt columns
    int sets;                 // sets of row-scale columns
    int resident;             // 1: the queries' scales stay in TMEM, 0: they are in the sets
    int smem;
};

struct TcParams {
    const float* row_scale;   // [n_rows]
    const float* q_scale;     // [query slot]
    int64_t n_rows;
    int nq;
    Plan plan;
    int mmas;                 // 64-element steps per tile
    int atoms;                // scale atoms per 128 rows
    int n_tiles;              // row tiles of this launch ...
    int tile_step;            // ... the j-th being tile j * tile_step, or with
    int tile_skip;            // tile_skip = r > 0 the j-th such tile with j not a multiple of r
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
    int test_stall;           // in the first pair a wait for a barrier nothing arrives on: 1 the
                              // issuer, 2 the second CTA's copies after a stage, 3 the first's
};

// ------------------------------------------------------------- PTX pieces --
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\t"
                 "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of a shared-memory object of a CTA of the pair, by rank.
__device__ __forceinline__ uint32_t smem_of(const void* p, uint32_t rank) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// Arrives on the first CTA's copy of a barrier.  Relaxed: what the arrival stands for is in TMEM
// (stores and loads that were waited for, ordered by the tcgen05 fences around the arrival and the
// wait for it) and no memory access that it would have to pass on; a release at cluster scope
// costs a fence per arrival.
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(smem_of(bar, 0))
                 : "memory");
}
// A copy into this CTA's shared memory that completes on the first CTA's copy of a barrier, so
// that the thread which waits there may let the tensor cores read both CTAs' shares.
__device__ __forceinline__ void tma_load_pair(void* smem_dst, const CUtensorMap* map, uint64_t* bar,
                                              int32_t x, int32_t y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_of(bar, 0))
        : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
// Counts bytes of a phase as arrived that no copy will bring.
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "r"(bytes)
                 : "memory");
}
// A value for both CTAs' copies of a word.
__device__ __forceinline__ void tell_pair(int* word, int value) {
#pragma unroll
    for (uint32_t r = 0; r < 2; ++r)
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(smem_of(word, r)), "r"(value) : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_slot, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(smem_slot)),
                 "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
                 : "memory");
}
// Arrives on both CTAs' copies of a barrier when the MMAs issued so far are done.
__device__ __forceinline__ void tc_commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

// One lane of the warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(one));
    return one != 0;
}

// Instruction descriptor of the block-scaled kinds: e2m1 x e2m1 -> f32, both K-major.
template <int FMT>
__host__ __device__ constexpr uint32_t make_idesc_fp4(int m, int n) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
           ((FMT == kMX ? 1u : 0u) << 23) | (static_cast<uint32_t>(m >> 4) << 24);
}

template <int FMT>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                        uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
    if (FMT == kMX)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X"
            " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X"
            " [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d_tmem),
            "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}

// This warp's lanes of consecutive columns of TMEM, four to a scale atom.
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint4 (&v)[2]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w)
                 : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint4 (&v)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(v[0].x), "r"(v[0].y), "r"(v[0].z), "r"(v[0].w), "r"(v[1].x), "r"(v[1].y), "r"(v[1].z), "r"(v[1].w), "r"(v[2].x), "r"(v[2].y), "r"(v[2].z), "r"(v[2].w), "r"(v[3].x), "r"(v[3].y), "r"(v[3].z), "r"(v[3].w)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
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

// One 32-column chunk of one row's scores, the first n of them, to out[t][col], t from t0.  NaN,
// which an empty row's or query's scale makes of a score, becomes -inf.  (A live row has none: an
// accumulator that has become infinite stays so, also where the other infinity is added.)
template <class T, bool FULL>
__device__ __forceinline__ void store_columns(const uint32_t (&r)[32], T* out, int64_t ld, int n,
                                              const float* gq, float g) {
    const float4* g4 = reinterpret_cast<const float4*>(gq);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 s = g4[i];
        const float x[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = 4 * i + u;
            if (FULL || j < n) {
                *out = cast_out<T>(fmaxf(__uint_as_float(r[j]) * g * x[u], -INFINITY));
                out += ld;
            }
        }
    }
}
template <class T>
__device__ __forceinline__ void store_chunk(const uint32_t (&r)[32], const TcParams& p, int t0,
                                            int n, int64_t col, const float* gq, float g) {
    T* out = static_cast<T*>(p.out) + (int64_t)t0 * p.ld + col;
    if (n == 32)
        store_columns<T, true>(r, out, p.ld, n, gq, g);
    else
        store_columns<T, false>(r, out, p.ld, n, gq, g);
}

// Candidates that an epilogue warp has found and not yet appended.  Their places in the queries'
// lists are asked for 32 at a time and used a tile later: the answer takes about as long as
// the MMAs of a third of a tile, and a pair waits for the last of its 32 warps.
struct Hits {
    uint64_t* entry;  // [HITS] score bits << 32 | row
    uint8_t* col;     // [HITS] query's column
    int n;            // warp-uniform
    int at;           // this lane's place, where asked for
    bool asked;       // for the first 32
};

__device__ __forceinline__ void ask_places(Hits& h, const TcParams& p, int qt_first, int lane) {
    __syncwarp();
    if (lane < h.n) h.at = atomicAdd(&p.cand_n[qt_first + h.col[lane]], 1);
    h.asked = true;
}

// The first 32 go to their places, the others move up.
__device__ __forceinline__ void place_hits(Hits& h, const TcParams& p, int qt_first, int lane) {
    __syncwarp();
    if (lane < h.n && h.at < CAP)
        p.cand[(int64_t)(qt_first + h.col[lane]) * CAP + h.at] = h.entry[lane];
    __syncwarp();
    if (lane + 32 < h.n) {
        h.entry[lane] = h.entry[lane + 32];
        h.col[lane] = h.col[lane + 32];
    }
    __syncwarp();
    h.n = max(h.n - 32, 0);
    h.asked = false;
}

// r[i], without an indexed access that would move r to local memory: a tree of selects.
__device__ __forceinline__ float pick(const uint32_t (&r)[32], int i) {
    uint32_t t[16];
    asm("{\n\t.reg .pred p;\n\t.reg .b32 x;\n\tand.b32 x, %48, 1;\n\tsetp.ne.u32 p, x, 0;\n\t"
        "selp.b32 %0, %17, %16, p;\n\t"
        "selp.b32 %1, %19, %18, p;\n\t"
        "selp.b32 %2, %21, %20, p;\n\t"
        "selp.b32 %3, %23, %22, p;\n\t"
        "selp.b32 %4, %25, %24, p;\n\t"
        "selp.b32 %5, %27, %26, p;\n\t"
        "selp.b32 %6, %29, %28, p;\n\t"
        "selp.b32 %7, %31, %30, p;\n\t"
        "selp.b32 %8, %33, %32, p;\n\t"
        "selp.b32 %9, %35, %34, p;\n\t"
        "selp.b32 %10, %37, %36, p;\n\t"
        "selp.b32 %11, %39, %38, p;\n\t"
        "selp.b32 %12, %41, %40, p;\n\t"
        "selp.b32 %13, %43, %42, p;\n\t"
        "selp.b32 %14, %45, %44, p;\n\t"
        "selp.b32 %15, %47, %46, p;\n\t}"
        : "=&r"(t[0]), "=&r"(t[1]), "=&r"(t[2]), "=&r"(t[3]), "=&r"(t[4]), "=&r"(t[5]), "=&r"(t[6]), "=&r"(t[7]), "=&r"(t[8]), "=&r"(t[9]), "=&r"(t[10]), "=&r"(t[11]), "=&r"(t[12]), "=&r"(t[13]), "=&r"(t[14]), "=&r"(t[15])
        : "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(i));
#pragma unroll
    for (int w = 8, b = 1; w >= 1; w /= 2, ++b) {
        const bool odd = (i >> b) & 1;
#pragma unroll
        for (int j = 0; j < w; ++j) t[j] = odd ? t[2 * j + 1] : t[2 * j];
    }
    return __uint_as_float(t[0]);
}

// One chunk of 32 columns of 32 rows, for the queries from column `at`: the rows that reach a
// query's threshold are kept.  Most chunks have none.  The sign of threshold - score is shifted
// into a mask (that of a NaN, an empty row's, is clear); then each lane deals with its own
// hits, one a round.
__device__ __forceinline__ void collect_chunk(const uint32_t (&r)[32], const TcParams& p, Hits& h,
                                              int qt_first, int at, int64_t row, const float* gq,
                                              const float* th, float g, int lane) {
    const float4* t4 = reinterpret_cast<const float4*>(th + at);
    const float minus_g = -g;
    uint32_t mine = 0;  // column i in bit 31 - i
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 t = t4[i];
        const float x[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
            mine = __funnelshift_l(
                __float_as_uint(fmaf(__uint_as_float(r[4 * i + u]), minus_g, x[u])), mine, 1);
    }
    unsigned lanes = __ballot_sync(0xffffffffu, mine != 0);
    while (lanes) {
        if (h.n > HITS - 32) {  // no room for a round
            if (!h.asked) ask_places(h, p, qt_first, lane);
            place_hits(h, p, qt_first, lane);
        }
        const int i = __clz((int)mine);
        const float v = pick(r, i) * g;
        if (mine) {
            const int slot = h.n + __popc(lanes & ((1u << lane) - 1u));
            h.entry[slot] = ((uint64_t)__float_as_uint(v * gq[at + i]) << 32) | (uint32_t)row;
            h.col[slot] = (uint8_t)(at + i);
            mine &= ~(0x80000000u >> i);
        }
        h.n += __popc(lanes);
        lanes = __ballot_sync(0xffffffffu, mine != 0);
    }
}

__device__ __forceinline__ int tile_of(const TcParams& p, int j) {
    return p.tile_step * (p.tile_skip > 0 ? j + j / (p.tile_skip - 1) + 1 : j);
}

// ------------------------------------------------------------ the product --
// A CTA pair works on tiles of 256 rows, 128 per CTA, against its tile of queries: each CTA
// keeps the codes of half of them in shared memory and streams its rows' codes and scales
// through a ring.  The codes of both CTAs complete on a barrier of the first, the scales on each
// CTA's own.  Scale warps move the scales into TMEM -- the rows' per stage into sets of columns used
// in turn, the queries' once where they fit (tcgen05.cp was tried first: its copies queue with the
// MMAs, about 90 ns each, and took longer than them) -- and arrive on the barrier of the codes, so
// that the issuing warp waits once a stage (on a barrier each for codes and scales, a batch's main
// pass took 3 % longer).
template <int FMT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    fp4_tc_kernel(const __grid_constant__ CUtensorMap tmap_rows,
                  const __grid_constant__ CUtensorMap tmap_row_sf,
                  const __grid_constant__ CUtensorMap tmap_q,
                  const __grid_constant__ CUtensorMap tmap_q_sf, const TcParams p, int mode) {
    constexpr int APS = atoms_per_stage(FMT);
    constexpr int STAGE = A_BYTES + APS * 512;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    // Both CTAs of a pair have the same shared-memory layout.
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                               ~static_cast<uintptr_t>(1023));
    const int nt = p.plan.nt, kchunks = p.plan.kchunks, stages = p.plan.stages;
    const int bufs = p.plan.bufs, sets = p.plan.sets;
    const bool resident = p.plan.resident != 0;
    const int sf_tiles = p.plan.nt_pad / 128;
    uint8_t* ring = smem;                                    // stages x (codes, scale atoms)
    uint8_t* sB = ring + stages * STAGE;                     // [kchunk][nt / 2][128 B], swizzled
    uint8_t* sSF = sB + kchunks * (nt / 2) * KC;             // [128-query tile][kchunk][APS]
    if (resident) sSF = ring;                                // ... only until it is in TMEM
    uint8_t* after = sB + kchunks * (nt / 2) * KC + (resident ? 0 : sf_tiles * kchunks * APS * 512);
    float* s_gq = reinterpret_cast<float*>(after);           // 16-byte aligned, like s_th
    float* s_th = s_gq + MAX_NT;
    uint64_t* s_hits = reinterpret_cast<uint64_t*>(s_th + MAX_NT);
    uint8_t* s_hit_col = reinterpret_cast<uint8_t*>(s_hits + EPI_WARPS * HITS);
    uint64_t* full = reinterpret_cast<uint64_t*>(s_hit_col + EPI_WARPS * HITS);  // a stage's scales
    uint64_t* ready = full + MAX_STAGES;     // on the first CTA: both CTAs' codes, and scales in TMEM
    uint64_t* empty = ready + MAX_STAGES;
    uint64_t* sfree = empty + MAX_STAGES;    // per set
    uint64_t* tfull = sfree + MAX_STAGES;
    uint64_t* tempty = tfull + 2;            // on the first CTA
    uint64_t* bfull = tempty + 2;            // the queries' scales
    uint64_t* bcodes = bfull + 1;            // on the first CTA: both CTAs' queries' codes
    uint64_t* qsf_done = bcodes + 1;
    uint64_t* drain = qsf_done + 1;
    uint64_t* stall = drain + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stall + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    // at the end, alike in both CTAs: whether every MMA was issued, and the stages that each CTA has
    // copied and each of its scale warps has put into TMEM
    int* finished = const_cast<int*>(abort_flag) + 1;
    int* copied = finished + 1;
    int* scaled = copied + 2;

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);  // warp-uniform
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1;
    const int qt = pair % p.plan.n_qt;
    const int stride = (gridDim.x >> 1) / p.plan.n_qt;  // pairs per query tile
    const int first = pair / p.plan.n_qt;
    // TMEM columns: accumulators, query scales (resident), sets of scales
    const uint32_t col_sfb = bufs * nt;
    const uint32_t set_cols = APS * 4 * (1 + (resident ? 0 : sf_tiles));
    const uint32_t col_sets = col_sfb + (resident ? sf_tiles * kchunks * APS * 4 : 0);

    if (threadIdx.x == 0) {
        for (int s = 0; s < MAX_STAGES; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&ready[s], 1 + 2 * SCALE_WARPS);
            mbar_init(&empty[s], 1 + SCALE_WARPS);
            mbar_init(&sfree[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], 2 * EPI_WARPS);
        }
        mbar_init(bfull, 1);
        mbar_init(bcodes, 1);
        mbar_init(qsf_done, SCALE_WARPS);
        mbar_init(drain, 1);
        mbar_init(stall, 1);
        *abort_flag = 0;
        *finished = 0;
        copied[0] = copied[1] = 0;
        fence_barrier_init();
    }
    if (warp == 5) tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    constexpr uint32_t tmem_base = 0;  // all 512 columns are this pair's
    // Up to here nothing of an earlier kernel's is read.
    griddep_launch();
    griddep_wait();
    for (int j = threadIdx.x; j < MAX_NT; j += THREADS) {
        const int t = qt * nt + j;
        const bool ok = j < nt && t < p.nq;
        s_gq[j] = ok ? __ldcg(p.q_scale + (int64_t)qt * p.plan.nt_pad + j) : 0.0f;
        s_th[j] = ok && mode == kCollect ? __ldcg(p.theta + t) : INFINITY;
    }
    __syncthreads();

    if (warp < SCALE_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_SCALE));
        // -------------------------------------------------------- scale warps
        const uint32_t lanes = tmem_base + ((uint32_t)(warp * 32) << 16);
        bool ok = __all_sync(0xffffffffu,
                             mbar_wait(bfull, 0, p.status, abort_flag, p.wait_ns));
        // A stage's scales of the queries, atom by atom the 128-query tiles side by side.
        auto put_queries = [&](uint32_t at, int kc) {
            const uint8_t* from = sSF + kc * APS * 512 + lane * 16;
            const int tile = kchunks * APS * 512;
            if (sf_tiles == 1) {
                uint4 v[APS];
#pragma unroll
                for (int a = 0; a < APS; ++a) v[a] = *reinterpret_cast<const uint4*>(from + a * 512);
                tmem_st(at, v);
            } else {
#pragma unroll
                for (int a = 0; a < APS; a += 2) {
                    uint4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[i] = *reinterpret_cast<const uint4*>(from + (i & 1) * tile +
                                                               (a + (i >> 1)) * 512);
                    tmem_st(at + a * 8, v);
                }
            }
        };
        if (ok && resident) {
            for (int kc = 0; kc < kchunks; ++kc)
                put_queries(lanes + col_sfb + kc * APS * sf_tiles * 4, kc);
            tmem_st_wait();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(qsf_done);
        int stage = 0, set = 0, done = 0;
        uint32_t phase = 0, set_phase = 0;
        for (int j = first; j < p.n_tiles && ok; j += stride) {
            for (int kc = 0; kc < kchunks; ++kc) {
                ok = __all_sync(0xffffffffu,
                                mbar_wait(&full[stage], phase, p.status, abort_flag, p.wait_ns));
                if (!ok) break;
                uint4 v[APS];
                const uint8_t* atoms = ring + stage * STAGE + A_BYTES;
#pragma unroll
                for (int a = 0; a < APS; ++a)
                    v[a] = *reinterpret_cast<const uint4*>(atoms + a * 512 + lane * 16);
                ok = __all_sync(0xffffffffu, mbar_wait(&sfree[set], set_phase ^ 1u, p.status,
                                                       abort_flag, p.wait_ns));
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = lanes + col_sets + set * set_cols;
                tmem_st(at, v);
                if (!resident) put_queries(at + APS * 4, kc);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_leader(&ready[stage]);
                    mbar_arrive(&empty[stage]);
                }
                ++done;
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
                if (++set == sets) {
                    set = 0;
                    set_phase ^= 1u;
                }
            }
        }
        if (lane == 0) tell_pair(&scaled[(int)rank * SCALE_WARPS + warp], done);
        __syncwarp();
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ISSUE));
        if (warp == 4 && lane == 0) {
            // -------------------------------------------------- TMA producer
            tma_prefetch_desc(&tmap_rows);
            tma_prefetch_desc(&tmap_row_sf);
            const int half_nt = nt / 2;
            mbar_arrive_expect_tx(bfull, (uint32_t)(sf_tiles * kchunks * APS * 512));
            if (rank == 0) mbar_arrive_expect_tx(bcodes, (uint32_t)(2 * kchunks * half_nt * KC));
            for (int kc = 0; kc < kchunks; ++kc) {
                tma_load_pair(sB + kc * half_nt * KC, &tmap_q, bcodes, kc * KC,
                              qt * p.plan.nt_pad + (int)rank * half_nt);
                for (int h = 0; h < sf_tiles; ++h)
                    tma_load_2d(sSF + (h * kchunks + kc) * APS * 512, &tmap_q_sf, bfull, 0,
                                (qt * sf_tiles + h) * p.atoms + kc * APS);
            }
            // The ring holds the queries' scales until they are in TMEM.
            bool ok = mbar_wait(qsf_done, 0, p.status, abort_flag, p.wait_ns);
            int stage = 0, loads = 0;
            uint32_t phase = 0, issued = 0, parity = 0;  // bits by stage
            for (int j = first; j < p.n_tiles && ok; j += stride) {
                const int half_tile = tile_of(p, j) * 2 + (int)rank;
                for (int kc = 0; kc < kchunks; ++kc) {
                    if (p.test_stall > 1 && pair == 0 && (int)rank == 3 - p.test_stall && loads == 1)
                        ok = mbar_wait(stall, 0, p.status, abort_flag, p.wait_ns);
                    if (!ok) break;
                    if (!mbar_wait(&empty[stage], phase ^ 1u, p.status, abort_flag, p.wait_ns)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = ring + stage * STAGE;
                    // (the other CTA's codes may land on the barrier before this arrival: its
                    // phase ends with it)
                    if (rank == 0) mbar_arrive_expect_tx(&ready[stage], 2 * A_BYTES);
                    mbar_arrive_expect_tx(&full[stage], APS * 512);
                    tma_load_pair(dst, &tmap_rows, &ready[stage], kc * KC, half_tile * HALF);
                    tma_load_2d(dst + A_BYTES, &tmap_row_sf, &full[stage], 0,
                                half_tile * p.atoms + kc * APS);
                    ++loads;
                    issued |= 1u << stage;
                    parity = (parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every copy this thread issued lands before the CTA may exit (a wait of its own
            // length: the caller's budget may have run out); the codes are waited for below.
            mbar_wait(bfull, 0, p.status, nullptr, kWaitBudgetNs);
            if (rank == 0) mbar_wait(bcodes, 0, p.status, nullptr, kWaitBudgetNs);
            for (int s = 0; s < stages; ++s)
                if ((issued >> s) & 1u)
                    mbar_wait(&full[s], (parity >> s) & 1u, p.status, nullptr, kWaitBudgetNs);
            tell_pair(&copied[rank], loads);
        } else if (warp == 5 && rank == 0) {
            // --------------------------------------------------- MMA issuer
            // The whole warp runs the loop, so that every operand is in a uniform register; one
            // lane issues.  (From a branch of one lane an MMA took 130 ns to issue, whatever
            // its shape.)
            const uint32_t idesc = make_idesc_fp4<FMT>(ROWS, nt);
            const uint64_t a_first = make_sw128_kmajor_desc(smem_u32(ring));
            const uint64_t b_first = make_sw128_kmajor_desc(smem_u32(sB));
            const uint32_t b_step = (uint32_t)(nt / 2) * KC >> 4;
            const bool one = elect_one();
            int stage = 0, set = 0, buf = 0;
            uint32_t phase = 0, buf_phase = 0;
            bool ok = p.test_stall != 1 || blockIdx.x != 0;
            if (!ok) mbar_wait(stall, 0, p.status, abort_flag, p.wait_ns);
            ok = ok && __all_sync(0xffffffffu,
                                  mbar_wait(bcodes, 0, p.status, abort_flag, p.wait_ns));
            for (int j = first; j < p.n_tiles && ok; j += stride) {
                ok = __all_sync(0xffffffffu, mbar_wait(&tempty[buf], buf_phase ^ 1u, p.status,
                                                       abort_flag, p.wait_ns));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * nt);
                for (int kc = 0; kc < kchunks; ++kc) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&ready[stage], phase, p.status,
                                                           abort_flag, p.wait_ns));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t a = a_first + (uint32_t)(stage * (STAGE >> 4));
                    const uint64_t b = b_first + (uint32_t)kc * b_step;
                    const uint32_t sfa = tmem_base + col_sets + set * set_cols;
                    const uint32_t sfb = resident
                                             ? tmem_base + col_sfb + kc * APS * sf_tiles * 4
                                             : sfa + APS * 4;
                    const bool whole = p.mmas - kc * 4 >= 4;  // else 128 elements, two steps
                    if (one) {
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            // MX: an atom's bytes 0-1 scale one 64-element step, 2-3 the next
                            constexpr bool mx = FMT == kMX;
                            const int atom = mx ? kk >> 1 : kk;
                            const uint32_t id = mx ? (uint32_t)(kk & 1) * 2u : 0u;
                            if (kk < 2 || whole)
                                mma_fp4<FMT>(d_tmem, a + kk * 2, b + kk * 2,
                                             idesc | (id << 4) | (id << 29), sfa + atom * 4,
                                             sfb + atom * sf_tiles * 4,
                                             kk == 0 ? (kc != 0 ? 1u : 0u) : 1u);
                        }
                        tc_commit_pair(&empty[stage]);
                        tc_commit_pair(&sfree[set]);
                        if (kc == kchunks - 1) tc_commit_pair(&tfull[buf]);
                    }
                    __syncwarp();
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (++set == sets) set = 0;
                }
                if (++buf == bufs) {
                    buf = 0;
                    buf_phase ^= 1u;
                }
            }
            // All MMAs issued above complete before TMEM is released.
            if (one) {
                tc_commit_pair(drain);
                tell_pair(finished, ok);
            }
            __syncwarp();
            mbar_wait(drain, 0, p.status, nullptr, kWaitBudgetNs);
        } else if (warp == 5) {
            // The other CTA stays until the last arrival on its barriers is in.
            mbar_wait(drain, 0, p.status, nullptr, kWaitBudgetNs);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_EPI));
        // ---------------------------------------------------------- epilogue
        const int quarter = warp & 3;
        const int half = (warp - 8) >> 2;      // of PER_QUARTER
        const int chunks = (nt + 31) / 32;     // of 32 columns; this warp takes every PER_QUARTER-th
        const int in_tile = (int)rank * HALF + quarter * 32 + lane;
        Hits hits = {s_hits + (warp - 8) * HITS, s_hit_col + (warp - 8) * HITS, 0, 0, false};
        int buf = 0;
        uint32_t buf_phase = 0;
        for (int j = first; j < p.n_tiles; j += stride) {
            const int64_t row = (int64_t)tile_of(p, j) * ROWS + in_tile;
            const bool row_in = row < p.n_rows;
            const float g = row_in ? __ldcg(&p.row_scale[row]) : __int_as_float(0x7fc00000);
            const bool got = mbar_wait(&tfull[buf], buf_phase, p.status, abort_flag, p.wait_ns);
            if (!__all_sync(0xffffffffu, got)) break;
            tc_fence_after();
            const uint32_t taddr =
                tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * nt);
            uint32_t r[HELD][32];
#pragma unroll
            for (int c = 0; c < HELD; ++c)
                if (PER_QUARTER * c + half < chunks)
                    tmem_ld32(taddr + (PER_QUARTER * c + half) * 32, r[c]);
#pragma unroll
            for (int c = 0; c < HELD; ++c) tmem_ld_wait_regs(r[c]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_leader(&tempty[buf]);
            const int64_t col = (int64_t)j * ROWS + in_tile;
#pragma unroll
            for (int c = 0; c < HELD; ++c) {
                const int at = (PER_QUARTER * c + half) * 32;
                if (at >= nt) break;
                if (mode == kCollect) {
                    collect_chunk(r[c], p, hits, qt * nt, at, row, s_gq, s_th, g, lane);
                    continue;
                }
                const int t0 = qt * nt + at;
                const int n = min(32, min(nt - at, p.nq - t0));
                if (!row_in || n <= 0) continue;
                if (p.out_type == PION_B200_F32)
                    store_chunk<float>(r[c], p, t0, n, col, s_gq + at, g);
                else if (p.out_type == PION_B200_BF16)
                    store_chunk<__nv_bfloat16>(r[c], p, t0, n, col, s_gq + at, g);
                else
                    store_chunk<__half>(r[c], p, t0, n, col, s_gq + at, g);
            }
            if (hits.asked) place_hits(hits, p, qt * nt, lane);
            if (hits.n >= 32) ask_places(hits, p, qt * nt, lane);
            if (++buf == bufs) {
                buf = 0;
                buf_phase ^= 1u;
            }
        }
        while (hits.n > 0) {
            if (!hits.asked) ask_places(hits, p, qt * nt, lane);
            place_hits(hits, p, qt * nt, lane);
        }
    }
    tc_fence_before();
    cluster_sync();
    if (!*finished) {
        // A wait ran out.  Codes may be on their way into either CTA, whose barriers lie in the
        // first: what one CTA has not copied of the stages that the other has, and what scale
        // warps have not put into TMEM, is made up for, then each stage's last phase waited for.
        // (Phases before it are complete: a stage is copied again once it has been multiplied.)
        if (rank == 0 && warp == 4 && lane == 0) {
            const int most = max(copied[0], copied[1]);
            for (int i = max(most - stages, 0); i < most; ++i) {
                uint64_t* bar = &ready[i % stages];
                if (i >= copied[0])
                    mbar_arrive_expect_tx(bar, A_BYTES);
                else if (i >= copied[1])
                    mbar_complete_tx(bar, A_BYTES);
                int missing = 0;
                for (int w = 0; w < 2 * SCALE_WARPS; ++w) missing += scaled[w] <= i;
                if (missing) mbar_arrive_n(bar, (uint32_t)missing);
                mbar_wait(bar, (uint32_t)(i / stages) & 1u, p.status, nullptr, kWaitBudgetNs);
            }
        }
        __syncwarp();
        cluster_sync();
    }
    if (warp == 5) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// --------------------------------------------------------------- selection --
constexpr int SEL = 256;  // threads of a selection CTA

__device__ __forceinline__ uint32_t ordered_score(float v) { return v == v ? ordered(v) : 0u; }

// The k-th largest of a warp's 32 V values, bit by bit from the highest: a bit is set if k values
// reach the number with it; once exactly k do, it is the least of those.  About 50 + 2 V
// cycles a bit, and no shared memory.
template <int V>
__device__ __forceinline__ uint32_t warp_kth(const uint32_t (&v)[V], int k) {
    uint32_t x = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
        const uint32_t y = x | (1u << b);
        constexpr int S = V < 4 ? V : 4;  // independent sums
        int part[S] = {};
#pragma unroll
        for (int i = 0; i < V; ++i) part[i % S] += v[i] >= y;
        int c = part[0];
#pragma unroll
        for (int i = 1; i < S; ++i) c += part[i];
        c = __reduce_add_sync(0xffffffffu, c);
        if (c >= k) x = y;
        if (c == k) break;
    }
    uint32_t least = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < V; ++i) least = v[i] >= x ? min(least, v[i]) : least;
    return __reduce_min_sync(0xffffffffu, least);
}

template <int V, class F>
__device__ __forceinline__ uint32_t warp_kth_of(int m, int k, F value) {
    const int lane = threadIdx.x & 31;
    uint32_t v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = lane + 32 * i < m ? value(lane + 32 * i) : 0u;
    return warp_kth<V>(v, k);
}

// The k-th largest of n <= LIST values in shared memory, by a CTA of NT threads: one warp's search of few,
// else the same search by all with a barrier a bit.
template <int NT>
__device__ uint32_t list_kth(const uint32_t* list, int n, int k) {
    constexpr int MOST = NT > 256 ? 32 : 16;  // values a lane holds
    __shared__ uint32_t s_kth;
    __shared__ int s_bit[32];
    if (n <= 32 * MOST) {
        if (threadIdx.x < 32) {
            auto at = [&](int i) { return list[i]; };
            const uint32_t x = n <= 64    ? warp_kth_of<2>(n, k, at)
                               : n <= 256 ? warp_kth_of<8>(n, k, at)
                                          : warp_kth_of<MOST>(n, k, at);
            if (threadIdx.x == 0) s_kth = x;
        }
        __syncthreads();
        return s_kth;
    }
    constexpr int V = LIST / NT;
    uint32_t v[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        v[i] = (int)threadIdx.x + i * NT < n ? list[threadIdx.x + i * NT] : 0u;
    if (threadIdx.x < 32) s_bit[threadIdx.x] = 0;
    __syncthreads();
    uint32_t x = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
        const uint32_t y = x | (1u << b);
        int c = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) c += v[i] >= y;
        c = __reduce_add_sync(0xffffffffu, c);
        if ((threadIdx.x & 31) == 0 && c) atomicAdd(&s_bit[b], c);
        __syncthreads();
        if (s_bit[b] >= k) x = y;
    }
    return x;
}

// The k-th largest (1-based, k <= 256, k <= m) of m ordered values, by a CTA of NT threads, or
// where more than LIST values reach it a lower bound of it.  Few values go through one warp;
// of more, the k-th largest of the threads' maxima is a lower bound that few values reach,
// and those are searched.  A thread keeps its first HOLD values in registers between the two
// passes.  `list` holds LIST values of scratch.
template <int NT, int HOLD, class F>
__device__ uint32_t kth_largest(int m, int k, uint32_t* list, F value) {
    __shared__ uint32_t s_low;
    __shared__ int s_count;
    if (m <= 512) {
        if (threadIdx.x < 32) {
            const uint32_t x = m <= 256 ? warp_kth_of<8>(m, k, value) : warp_kth_of<16>(m, k, value);
            if (threadIdx.x == 0) s_low = x;
        }
        __syncthreads();
        return s_low;
    }
    uint32_t held[HOLD];
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        const int i = threadIdx.x + h * NT;
        held[h] = i < m ? value(i) : 0u;
    }
#pragma unroll
    for (int h = 0; h < HOLD; ++h) top = max(top, held[h]);
    // four loads in flight at a time
    auto rest = [&](auto use) {
        for (int i = threadIdx.x + HOLD * NT; i < m; i += 4 * NT) {
            uint32_t o[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) o[u] = i + u * NT < m ? value(i + u * NT) : 0u;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i + u * NT < m) use(o[u]);
        }
    };
    rest([&](uint32_t o) { top = max(top, o); });
    list[threadIdx.x] = top;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        const uint32_t x = warp_kth_of<NT / 32>(NT, k, [&](int i) { return list[i]; });
        if (threadIdx.x == 0) s_low = x;
    }
    __syncthreads();
    const uint32_t low = s_low;
    auto keep = [&](uint32_t o) {
        const int at = atomicAdd(&s_count, 1);
        if (at < LIST) list[at] = o;
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h)
        if ((int)threadIdx.x + h * NT < m && held[h] >= low) keep(held[h]);
    rest([&](uint32_t o) {
        if (o >= low) keep(o);
    });
    __syncthreads();
    const int n = s_count;
    return n > LIST ? low : list_kth<NT>(list, n, k);
}

// A number that at least k, and few more, of n <= LIST values in shared memory reach: their k-th
// largest where a warp can hold them, else that of the maxima of groups of them.
template <int NT>
__device__ uint32_t list_low(const uint32_t* list, int n, int k) {
    __shared__ uint32_t s_low;
    if (threadIdx.x < 32) {
        uint32_t x;
        if (n <= 256) {
            x = warp_kth_of<8>(n, k, [&](int i) { return list[i]; });
        } else {
            // 16 groups a lane: more than k of them, of at most four values
            x = warp_kth_of<16>(512, k, [&](int i) {
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < LIST / 512; ++j)
                    top = i + 512 * j < n ? max(top, list[i + 512 * j]) : top;
                return top;
            });
        }
        if (threadIdx.x == 0) s_low = x;
    }
    __syncthreads();
    return s_low;
}

// Sorts n <= LIST keys in shared memory, largest first: up to a key per thread by their ranks,
// more by a bitonic sort over the next power of two (the rest is filled with zeros).
template <int NT>
__device__ void sort_desc(uint64_t* key, int n) {
    __syncthreads();
    if (n <= NT && n <= 512) {
        const int i = threadIdx.x;
        int at = 0;
        const uint64_t x = i < n ? key[i] : 0;
        if (i < n)
            for (int j = 0; j < n; ++j) {
                const uint64_t y = key[j];
                at += y > x || (y == x && j < i);
            }
        __syncthreads();
        if (i < n) key[at] = x;
        __syncthreads();
        return;
    }
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += NT) key[i] = 0;
    __syncthreads();
    for (int w = 2; w <= size; w <<= 1)
        for (int s = w >> 1; s; s >>= 1) {
            for (int i = threadIdx.x; i < size / 2; i += NT) {
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

// Infinite where a float32 sum, or its product with the row's g alone (a score in units of the
// query's g), could overflow: nothing is known of an approximate score then.  The last term
// covers products below the least normal float.
__device__ __forceinline__ float eps_of(int dp, float q_norm, float gq, float norm_max) {
    const float size = q_norm * norm_max, in_units = q_norm / gq * norm_max;
    return size < 0x1p120f && in_units < 0x1p120f ? rel_eps(dp) * size + 0x1p-100f : INFINITY;
}

// A query's threshold: the k-th best (ordered) of its approximate scores so far less 2 eps, in
// units of the query's g.
__device__ __forceinline__ float threshold_of(uint32_t kth, float two_eps, float gq) {
    const float x = ((kth ? unordered(kth) : -INFINITY) - two_eps) / gq;
    return x > -INFINITY ? x - 0x1p-20f * fabsf(x) : -INFINITY;
}

// First thresholds, one query per CTA, from the scores of 4 V4 NT sampled rows, which stay in
// registers: the k-th largest of the maxima of 256 groups of threads bounds the k-th best
// from below, and the few scores that reach it are searched.  Resets the candidate counts.
template <int NT, int V4>
__global__ void __launch_bounds__(NT)
    theta_sample_kernel(const float* sample, int k, int dp,
                        const float* q_scale, int nt, int nt_pad,
                        const float* q_norm, const float* norm_max,
                        float* theta, int* cand_n) {
    __shared__ uint32_t list[LIST];
    __shared__ uint32_t s_low;
    __shared__ int s_count;
    griddep_launch();
    griddep_wait();
    const int t = blockIdx.x;
    const float4* s = reinterpret_cast<const float4*>(sample) + (int64_t)t * NT * V4;
    float4 v[V4];
#pragma unroll
    for (int i = 0; i < V4; ++i) v[i] = __ldcg(s + threadIdx.x + i * NT);
    const float gq = __ldcg(q_scale + query_slot(t, nt, nt_pad));
    const float two_eps = 2.0f * eps_of(dp, __ldcg(q_norm + t), gq, __ldcg(norm_max));
    float most = -INFINITY;  // (passes over NaN)
#pragma unroll
    for (int i = 0; i < V4; ++i)
        most = fmaxf(most, fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w)));
#pragma unroll
    for (int o = 1; o < NT / 256; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    if (threadIdx.x % (NT / 256) == 0) list[threadIdx.x / (NT / 256)] = ordered(most);
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        const uint32_t x = warp_kth_of<8>(256, k, [&](int i) { return list[i]; });
        if (threadIdx.x == 0) s_low = x;
    }
    __syncthreads();
    const uint32_t low = s_low;
    const float low_f = unordered(low);
    // For small k hardly two of the k best share a group: the bound does.
    const bool near = k <= 32;
    auto keep = [&](float x) {
        if (x >= low_f) {
            const int at = atomicAdd(&s_count, 1);
            if (at < LIST) list[at] = ordered(x);
        }
    };
    uint32_t x = low;
    if (!near) {
#pragma unroll
        for (int i = 0; i < V4; ++i) {
            keep(v[i].x);
            keep(v[i].y);
            keep(v[i].z);
            keep(v[i].w);
        }
        __syncthreads();
        const int n = s_count;
        if (n <= LIST) x = list_kth<NT>(list, n, k);
    }
    if (threadIdx.x == 0) {
        // an empty or zero query collects nothing
        theta[t] = gq > 0.0f ? threshold_of(x, two_eps, gq) : INFINITY;
        cand_n[t] = 0;
    }
}

// Tighter thresholds, one query per CTA, from the candidates so far.
__global__ void __launch_bounds__(SEL)
    theta_kernel(const uint64_t* cand, int k, int dp, const float* q_scale, int nt, int nt_pad,
                 const float* q_norm, const float* norm_max, float* theta, const int* cand_n) {
    __shared__ uint32_t list[LIST];
    griddep_launch();
    griddep_wait();
    const int t = blockIdx.x;
    const int m = min(__ldcg(cand_n + t), CAP);
    const float gq = __ldcg(q_scale + query_slot(t, nt, nt_pad));
    const float two_eps = 2.0f * eps_of(dp, __ldcg(q_norm + t), gq, __ldcg(norm_max));
    if (!(gq > 0.0f) || m < k) return;
    const uint64_t* c = cand + (int64_t)t * CAP;
    const uint32_t x = kth_largest<SEL, 4>(m, k, list, [&](int i) {
        return ordered_score(__uint_as_float((uint32_t)(__ldcg(c + i) >> 32)));
    });
    if (threadIdx.x == 0) theta[t] = threshold_of(x, two_eps, gq);
}

// Few queries: the candidates straight from the scores of every row, a chunk of SPLIT rows per
// CTA.  A row among the k best overall is among the k best of its chunk, so its approximate
// score is at least the chunk's k-th best less 2 eps; for that the k-th largest of the
// threads' maxima does, a lower bound of it that few scores reach.
constexpr int SPLIT = 8192;
__global__ void __launch_bounds__(SEL)
    split_kernel(const float* scores, int64_t ld, int64_t n_rows, int k, int dp,
                 const float* q_scale, int nt, int nt_pad, const float* q_norm,
                 const float* norm_max, uint64_t* cand, int* cand_n) {
    constexpr int V4 = SPLIT / SEL / 4;
    __shared__ uint32_t list[SEL];
    __shared__ float s_cut;
    __shared__ int s_count, s_base;
    __shared__ uint64_t s_cand[LIST];
    griddep_launch();
    griddep_wait();
    const int t = blockIdx.y;
    const int64_t first = (int64_t)blockIdx.x * SPLIT;
    const float* s = scores + (int64_t)t * ld + first;
    const int64_t left = n_rows - first;
    float4 v[V4];
#pragma unroll
    for (int i = 0; i < V4; ++i) {  // ld is a multiple of 4: whole vectors lie inside the row
        const int at = 4 * (int)(threadIdx.x + i * SEL);
        v[i] = at < left ? __ldcg(reinterpret_cast<const float4*>(s + at))
                         : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at + 1 >= left) v[i].y = -INFINITY;
        if (at + 2 >= left) v[i].z = -INFINITY;
        if (at + 3 >= left) v[i].w = -INFINITY;
    }
    const float gq = __ldcg(q_scale + query_slot(t, nt, nt_pad));
    const float two_eps = 2.0f * eps_of(dp, __ldcg(q_norm + t), gq, __ldcg(norm_max));
    float most = -INFINITY;
#pragma unroll
    for (int i = 0; i < V4; ++i)
        most = fmaxf(most, fmaxf(fmaxf(v[i].x, v[i].y), fmaxf(v[i].z, v[i].w)));
    list[threadIdx.x] = ordered(most);
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    if (threadIdx.x < 32) {
        const uint32_t x = warp_kth_of<8>(SEL, k, [&](int i) { return list[i]; });
        if (threadIdx.x == 0) s_cut = unordered(x) - two_eps;
    }
    __syncthreads();
    if (!(gq > 0.0f)) return;  // an empty or zero query collects nothing
    const float cut = s_cut;
    auto keep = [&](float x, int at) {
        if (x >= cut && x > -INFINITY) {
            const int to = atomicAdd(&s_count, 1);
            if (to < LIST)
                s_cand[to] = ((uint64_t)__float_as_uint(x) << 32) | (uint32_t)(first + at);
        }
    };
#pragma unroll
    for (int i = 0; i < V4; ++i) {
        const int at = 4 * (int)(threadIdx.x + i * SEL);
        keep(v[i].x, at);
        keep(v[i].y, at + 1);
        keep(v[i].z, at + 2);
        keep(v[i].w, at + 3);
    }
    __syncthreads();
    // more than LIST in one chunk overflow the query's list: the rescue's to answer
    if (threadIdx.x == 0) s_base = atomicAdd(cand_n + t, s_count > LIST ? CAP + 1 : s_count);
    __syncthreads();
    const int n = min(s_count, LIST);
    for (int i = threadIdx.x; i < n; i += SEL)
        if (s_base + i < CAP) cand[(int64_t)t * CAP + s_base + i] = s_cand[i];
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
    int nq;
    int* n_flagged;          // queries left to rescue_kernel, their number
    int* flagged;            // ... which [nq]
    int* done;               // ... their finished parts [nq]
    uint64_t* parts;         // ... the parts' best keys [items][k]
    int32_t* out_ids;        // [nq][k]
    float* out_scores;
};

// The query's codes as bytes (twice their value); its block scales in units of 2^-9 (NV), or their
// exponents (MX).
struct QueryShared {
    int8_t* codes;
    uint32_t* scales;
};

constexpr long long kMantissa = (1ll << 52) - 1;  // of a float64

// 2^e as a float64, -1022 <= e <= 1023.
__device__ __forceinline__ double power_of_two(int e) { return __hiloint2double((e + 1023) << 20, 0); }

// A sum of products in units of both rows' g: m 2^e exactly, or where |m| has its highest bit at 61,
// m 2^e towards zero with the last bit set for what is left out.
struct Sum {
    long long m;
    int e;
};

// sum of q_j v_j over the block of 32 elements `raw`, four times over, in halves.
__device__ __forceinline__ void block_dots(const uint4& w, const int8_t* q, int (&dot)[2]) {
    const uint32_t raw[4] = {w.x, w.y, w.z, w.w};
    const int4* qb = reinterpret_cast<const int4*>(q);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int4 qq = qb[h];
        dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h]), qq.x, 0);
        dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h] >> 16), qq.y, dot[h]);
        dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h + 1]), qq.z, dot[h]);
        dot[h] = __dp4a((int)e2m1x4_bytes(raw[2 * h + 1] >> 16), qq.w, dot[h]);
    }
}

// MX sums whose blocks' exponents lie far apart, by half a warp: an integer of 16 digits of 32 bits
// (and a carry), a lane's digit the sum of those blocks' products that begin in it.
__device__ __noinline__ Sum half_warp_far_dot(const uint4* codes, const uint8_t* scales,
                                              const int8_t* q_codes, const uint32_t* q_scales,
                                              int blocks, int sub) {
    long long digit = 0;  // at most 256 blocks of 13 bits and 31: 53 bits
    for (int b0 = 0; b0 < blocks; b0 += 16) {
        const int b = b0 + sub;
        int dot[2] = {0, 0}, e = 0;
        if (b < blocks) {
            block_dots(__ldcg(codes + b), q_codes + b * 32, dot);
            e = (int)(q_scales[b] + __ldcg(scales + (b >> 2) * 512 + (b & 3)));  // 0 to 504
        }
        const int mine = dot[0] + dot[1];
        for (int i = 0; i < 16; ++i) {
            const int d = __shfl_sync(0xffffffffu, mine, i, 16);
            const int at = __shfl_sync(0xffffffffu, e, i, 16);
            if (at >> 5 == sub) digit += (long long)d << (at & 31);
        }
    }
    // The sign, then the magnitude's digits, from the lowest.
    bool negative = false;
    uint32_t d = 0, top = 0;
    for (int pass = 0; pass < 2; ++pass) {
        long long carry = 0;
        for (int i = 0; i < 16; ++i) {
            const long long x = __shfl_sync(0xffffffffu, digit, i, 16) + carry;
            if (i == sub) d = (uint32_t)x;
            carry = x >> 32;
        }
        top = (uint32_t)carry;
        if (pass == 0) {
            negative = carry < 0;
            if (negative) digit = -digit;
        }
    }
    // The highest digit that is not zero (the carry is the 17th), and the two below it.
    const unsigned half = (threadIdx.x & 16) ? 16 : 0;
    const unsigned some = (__ballot_sync(0xffffffffu, d != 0) >> half) & 0xFFFFu;
    const int h = top ? 16 : some ? 31 - __clz((int)some) : 0;
    const uint32_t d0 = __shfl_sync(0xffffffffu, d, h & 15, 16);
    const uint32_t d1 = __shfl_sync(0xffffffffu, d, (h - 1) & 15, 16);
    const uint32_t d2 = __shfl_sync(0xffffffffu, d, (h - 2) & 15, 16);
    const uint32_t a = h == 16 ? top : d0, b = h >= 1 ? d1 : 0u, c = h >= 2 ? d2 : 0u;
    if (a == 0) return {0, 0};
    const bool below = h >= 3 && (some & ((1u << (h - 2)) - 1u)) != 0;
    const int z = __clz((int)a);
    uint64_t m = ((uint64_t)a << 32 | b) << z;
    if (z) m |= c >> (32 - z);
    const bool rest = (uint32_t)(c << z) != 0 || below;  // (z < 32)
    m = m >> 2 | ((m & 3u) != 0 || rest ? 1u : 0u);
    // the digits' unit is 2^-256: a quarter of 2^-254
    return {negative ? -(long long)m : (long long)m, 32 * (h - 1) - z + 2 - 256};
}

// sum_j q_j v_j by half a warp (`sub`: the lane's place in it), in all its lanes.  NV: in units of
// 2^-20 a block's sum has at most 48 bits and a row's 57, an integer.  MX: a block's sum is an integer
// of 13 bits times a power of two; where those of a row are at most 2^32 apart, any order of them adds
// up in float64 without rounding.  A lane's loads of 64 blocks of 32 elements are in flight together.
template <int FMT>
__device__ __forceinline__ Sum half_warp_dot(const FinishParams& p, const QueryShared& q, int64_t row,
                                             int sub) {
    static_assert(kMaxDim / 32 * (36 * 4 * 32) <= 1 << 21, "53 bits");
    const uint4* codes = reinterpret_cast<const uint4*>(p.codes + row * (p.dp / 2));
    const uint8_t* scales = p.scales + scale_word(row, 0, p.atoms);
    const int blocks = p.dp / 32;
    double acc = 0.0;
    uint32_t reach = 0;  // the highest exponent, and 511 less the lowest
    long long sum = 0;
    for (int b0 = sub; b0 < blocks; b0 += 64) {
        uint4 w[4];
        uint32_t s[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int b = b0 + 16 * u;
            const bool in = b < blocks;
            w[u] = in ? __ldcg(codes + b) : make_uint4(0u, 0u, 0u, 0u);
            if (FMT == kMX)
                s[u] = in ? __ldcg(scales + (b >> 2) * 512 + (b & 3)) : 0u;
            else
                s[u] = in ? __ldcg(reinterpret_cast<const uint16_t*>(
                                scales + (b >> 1) * 512 + (b & 1) * 2))
                          : 0u;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int b = b0 + 16 * u;
            if (b >= blocks) break;
            int dot[2];
            block_dots(w[u], q.codes + b * 32, dot);
            if (FMT == kMX) {
                const uint32_t e = q.scales[b] + s[u];
                const int d = dot[0] + dot[1];
                acc = fma((double)d, power_of_two((int)e - 254), acc);
                if (d != 0) reach = __vmaxu2(reach, e << 16 | (511u - e));
            } else {
                sum += (long long)(dot[0] * (int)e4m3_units(s[u] & 255u)) * (int)q.scales[2 * b];
                sum += (long long)(dot[1] * (int)e4m3_units(s[u] >> 8)) * (int)q.scales[2 * b + 1];
            }
        }
    }
    if constexpr (FMT == kMX) {
#pragma unroll
        for (int o = 8; o; o >>= 1) {
            acc += __shfl_xor_sync(0xffffffffu, acc, o);
            reach = __vmaxu2(reach, __shfl_xor_sync(0xffffffffu, reach, o));
        }
        const bool far = (int)(reach >> 16) + (int)(reach & 0xFFFFu) - 511 > 32;
        if (__any_sync(0xffffffffu, far)) {
            const Sum x = half_warp_far_dot(codes, scales, q.codes, q.scales, blocks, sub);
            if (far) return x;
        }
        const long long bits = __double_as_longlong(acc);
        const int exponent = (int)(bits >> 52) & 0x7FF;  // at least 1023 - 254 where acc is not 0
        const long long m = exponent ? (bits & kMantissa) | 1ll << 52 : 0;
        return {bits < 0 ? -m : m, exponent - 1075 - 2};
    } else {
#pragma unroll
        for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return {sum, -20};
    }
}

// ((m 2^e) g_r) g_t, rounded once to float32.  The two scales' product has 48 bits: a float64.  The
// whole is rounded to the 53 bits of one with its last bit set for what is left out, so that the
// rounding to float32 is that of the exact product.
__device__ __forceinline__ float exact_score(Sum x, float g, float gq) {
    const double scale = (double)g * (double)gq;
    if (x.m == 0 || !(fabs(scale) > 0.0)) return (float)(scale * 0.0);  // (NaN for a NaN)
    const uint64_t a = (uint64_t)(x.m < 0 ? -x.m : x.m);
    if (a <= 1ull << 53) {
        const double v = (double)x.m * power_of_two(x.e);
        const double y = v * scale, left = fma(v, scale, -y);
        long long bits = __double_as_longlong(y);
        if (left != 0.0) bits = (bits - ((left > 0.0) != (y > 0.0))) | 1;
        return (float)__longlong_as_double(bits);
    }
    const long long bits = __double_as_longlong(scale);
    const uint64_t f = (uint64_t)((bits & kMantissa) | 1ll << 52) >> 5;
    const uint64_t hi = __umul64hi(a, f), lo = a * f;  // 2^100 to 2^110
    const int n = 64 - __clzll((long long)hi);
    const uint64_t top = hi << (64 - n) | lo >> n;
    const bool rest = lo << (64 - n) != 0 || (top & 0x7FFu) != 0;
    const double v = (double)(long long)(top >> 11 | (rest ? 1u : 0u)) *
                     power_of_two(x.e + ((int)(bits >> 52) & 0x7FF) - 1075 + 5 + n + 11);
    return (float)((x.m < 0) != (bits < 0) ? -v : v);
}

// Larger is better: (score desc, row asc); 0 for a row that cannot be found.
__device__ __forceinline__ uint64_t row_key(Sum dot, float g, float gq, int64_t row) {
    const float s = exact_score(dot, g, gq) + 0.0f;
    if (!(s > -INFINITY)) return 0;
    return ((uint64_t)ordered(s) << 32) | (uint32_t)~(uint32_t)row;
}

// By NT threads, this one the `at`-th.
template <int FMT, int NT>
__device__ __forceinline__ void load_query(const FinishParams& p, const QueryShared& q, int64_t qs,
                                           int at) {
    const uint16_t* codes = reinterpret_cast<const uint16_t*>(p.q_codes + qs * (p.dp / 2));
    for (int i = at; i < p.dp / 4; i += NT)
        reinterpret_cast<uint32_t*>(q.codes)[i] = e2m1x4_bytes(__ldcg(codes + i));
    for (int b = at; b < p.dp / block_of(FMT); b += NT) {
        const uint32_t byte = __ldcg(p.q_scales + scale_word(qs, b >> 2, p.atoms) + (b & 3));
        q.scales[b] = FMT == kMX ? byte : e4m3_units(byte);
    }
}

template <int NT>
__device__ __forceinline__ void write_best(const FinishParams& p, int t, const uint64_t* key,
                                           int found) {
    for (int j = threadIdx.x; j < p.k; j += NT) {
        const uint64_t x = j < found ? key[j] : 0;
        p.out_ids[(int64_t)t * p.k + j] =
            x ? (int32_t)(p.id_base + (int64_t)(uint32_t)~(uint32_t)x) : -1;
        p.out_scores[(int64_t)t * p.k + j] = x ? unordered((uint32_t)(x >> 32)) : -INFINITY;
    }
}

// The k best of a stream of keys, by a CTA: offered keys above the k-th best so far are kept
// until the list is nearly full, then the k best of them.
template <int NT>
struct BestKeys {
    static constexpr int BATCH = 512;  // offered at most between two calls of settle()
    uint64_t* key;                     // [LIST], shared
    int* n;                            // shared, 0 at first
    uint64_t floor;
    __device__ __forceinline__ void offer(uint64_t x) {  // by any thread
        if (x > floor) key[atomicAdd(n, 1)] = x;
    }
    __device__ __forceinline__ int settle(int k, bool last) {  // by all threads
        __syncthreads();
        int have = *n;
        if (have > LIST - BATCH || last) {
            sort_desc<NT>(key, have);
            have = min(have, k);
            floor = have == k ? key[k - 1] : 0;
            __syncthreads();
            if (threadIdx.x == 0) *n = have;
        }
        __syncthreads();
        return have;
    }
};

// The k best of rows [begin, end), all scored exactly, by a CTA -> key[0, found).  `n`: shared.
template <int FMT, int NT>
__device__ int scan_rows(const FinishParams& p, const QueryShared& q, float gq, int64_t begin,
                         int64_t end, uint64_t* key, int* n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int W = NT / 32, BATCH = BestKeys<NT>::BATCH;
    __syncthreads();
    if (threadIdx.x == 0) *n = 0;
    __syncthreads();
    BestKeys<NT> best = {key, n, 0};
    int found = begin < end ? 0 : best.settle(p.k, true);
    for (int64_t r0 = begin; r0 < end; r0 += BATCH) {
        for (int i = 2 * warp; i < BATCH && r0 + i < end; i += 2 * W) {
            const int64_t row = min(r0 + i + (lane >> 4), end - 1);
            const float g = __ldcg(p.row_scale + row);
            const Sum dot = half_warp_dot<FMT>(p, q, row, lane & 15);
            if ((lane & 15) == 0 && row == r0 + i + (lane >> 4))
                best.offer(row_key(dot, g, gq, row));
        }
        found = best.settle(p.k, r0 + BATCH >= end);
    }
    return found;
}

// The k best rows of one query per CTA: its candidates whose approximate score can be among
// the k best are scored exactly and sorted.  A query with more than LIST of those, or whose
// candidates overflowed, is left to rescue_kernel, or where all rows are few (dense) scored
// here row by row.
template <int FMT, int NT>
__global__ void __launch_bounds__(NT, NT > 256 ? 1 : 4) finish_kernel(const FinishParams p) {
    __shared__ __align__(16) uint64_t key[LIST];
    __shared__ int s_warp[NT / 32];
    __shared__ int s_n;
    extern __shared__ __align__(16) uint8_t dyn[];  // query bytes [dp], scales [dp / block]
    griddep_launch();
    griddep_wait();
    const int t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int W = NT / 32;
    const int64_t qs = query_slot(t, p.nt, p.nt_pad);
    // Every load that does not wait for another: the candidates' places, however many there are.
    constexpr int V = LIST / NT;
    const uint64_t* cand = p.cand + (int64_t)t * CAP;
    uint64_t c[V];
#pragma unroll
    for (int u = 0; u < V; ++u) c[u] = p.dense ? 0 : __ldcg(cand + threadIdx.x + u * NT);
    const float gq = __ldcg(p.q_scale + qs);
    const int m = p.dense ? (int)p.n_rows : __ldcg(p.cand_n + t);
    const float two_eps = 2.0f * eps_of(p.dp, __ldcg(p.q_norm + t), gq, __ldcg(p.norm_max));
    QueryShared q;
    q.codes = reinterpret_cast<int8_t*>(dyn);
    q.scales = reinterpret_cast<uint32_t*>(dyn + p.dp);
    if (warp > 0) load_query<FMT, NT - 32>(p, q, qs, threadIdx.x - 32);
    if (threadIdx.x == 0) s_n = 0;

    int found = 0;
    if (gq > 0.0f) {
        const bool known = two_eps < INFINITY;  // else any row may be among the best
        bool whole = !p.dense && (m > CAP || !known);
        if (!whole) {
            const float* dense = p.dense + (int64_t)t * p.ld;
            auto approx = [&](int i) {
                return p.dense ? __ldcg(dense + i)
                               : __uint_as_float((uint32_t)(__ldcg(cand + i) >> 32));
            };
            uint32_t* list = reinterpret_cast<uint32_t*>(key);
            // (-inf is an empty slot's: where the margin is known, no score of a row left float32)
            auto take = [&](float a, float cut, uint64_t row) {
                if ((a >= cut && a > -INFINITY) || !known) {
                    const int at = atomicAdd(&s_n, 1);
                    if (at < LIST) key[at] = row;
                }
            };
            auto cut_of = [&](uint32_t o) { return o ? unordered(o) - two_eps : -INFINITY; };
            if (!p.dense && m <= LIST) {
#pragma unroll
                for (int u = 0; u < V; ++u) {
                    const int i = threadIdx.x + u * NT;
                    if (i < m) list[i] = ordered_score(__uint_as_float((uint32_t)(c[u] >> 32)));
                }
                __syncthreads();
                const float cut = m <= p.k ? -INFINITY : cut_of(list_low<NT>(list, m, p.k));
                __syncthreads();
#pragma unroll
                for (int u = 0; u < V; ++u)
                    if ((int)threadIdx.x + u * NT < m)
                        take(__uint_as_float((uint32_t)(c[u] >> 32)), cut, c[u] & 0xFFFFFFFFu);
            } else {
                __syncthreads();
                float cut = -INFINITY;
                if (m > p.k)
                    cut = cut_of(kth_largest<NT, 8>(
                        m, p.k, list, [&](int i) { return ordered_score(approx(i)); }));
                __syncthreads();
                for (int i0 = threadIdx.x; i0 < m; i0 += 4 * NT) {
                    float a[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) a[u] = i0 + u * NT < m ? approx(i0 + u * NT) : 0.0f;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int i = i0 + u * NT;
                        if (i < m)
                            take(a[u], cut, p.dense ? (uint64_t)i : (__ldcg(cand + i) & 0xFFFFFFFFu));
                    }
                }
            }
            __syncthreads();
            whole = s_n > LIST;
            if (!whole) {
                for (int i0 = 2 * warp; i0 < s_n; i0 += 2 * W) {
                    const int i = min(i0 + (lane >> 4), s_n - 1);
                    const int64_t row = (int64_t)key[i];
                    const float g = __ldcg(p.row_scale + row);
                    const Sum dot = half_warp_dot<FMT>(p, q, row, lane & 15);
                    // (an odd one out is done by both halves, and written by the first)
                    if ((lane & 15) == 0 && i == i0 + (lane >> 4)) key[i] = row_key(dot, g, gq, row);
                }
                __syncthreads();
                found = s_n;
                sort_desc<NT>(key, found);
            }
        }
        if (whole && p.dense) {
            found = scan_rows<FMT, NT>(p, q, gq, 0, p.n_rows, key, &s_n);
        } else if (whole) {
            if (threadIdx.x == 0) {
                p.done[t] = 0;
                p.flagged[atomicAdd(p.n_flagged, 1)] = t;
            }
            return;
        }
    } else if (gq == 0.0f) {
        // Every row that holds anything scores 0: the first k of them.
        for (int64_t r0 = 0; r0 < p.n_rows && found < p.k; r0 += NT) {
            const int64_t row = r0 + threadIdx.x;
            const float g = row < p.n_rows ? __ldcg(p.row_scale + row) : __int_as_float(0x7fc00000);
            const unsigned live = __ballot_sync(0xffffffffu, g == g);
            if (lane == 0) s_warp[warp] = __popc(live);
            __syncthreads();
            int at = found;
            int all = 0;
            for (int w = 0; w < W; ++w) {
                if (w < warp) at += s_warp[w];
                all += s_warp[w];
            }
            at += __popc(live & ((1u << lane) - 1u));
            if (g == g && at < p.k) key[at] = ((uint64_t)ordered(0.0f) << 32) | (uint32_t)~(uint32_t)row;
            found += all;
            __syncthreads();
        }
    }
    __syncthreads();
    write_best<NT>(p, t, key, found);
}

// Flagged queries (many rows that tie with the k-th best, a sample that missed the best rows, or
// norms whose products leave float32) of many rows: every row, exactly.  Each query's rows are split
// between as many CTAs as the grid has to spare; the last one to finish merges the parts.
constexpr int RESCUE_CTAS = 296;
template <int FMT>
__global__ void __launch_bounds__(SEL) rescue_kernel(const FinishParams p) {
    __shared__ __align__(16) uint64_t key[LIST];
    __shared__ int s_n;
    __shared__ int s_last;
    extern __shared__ __align__(16) uint8_t dyn[];
    griddep_launch();
    griddep_wait();
    const int flagged = __ldcg(p.n_flagged);
    if (flagged == 0) return;
    QueryShared q;
    q.codes = reinterpret_cast<int8_t*>(dyn);
    q.scales = reinterpret_cast<uint32_t*>(dyn + p.dp);
    const int splits = max(1, RESCUE_CTAS / flagged);
    for (int item = blockIdx.x; item < flagged * splits; item += gridDim.x) {
        const int t = __ldcg(p.flagged + item / splits);
        const int part = item % splits;
        const int64_t qs = query_slot(t, p.nt, p.nt_pad);
        const float gq = __ldcg(p.q_scale + qs);
        const int64_t begin = p.n_rows * part / splits, end = p.n_rows * (part + 1) / splits;
        load_query<FMT, SEL>(p, q, qs, threadIdx.x);
        int found = scan_rows<FMT, SEL>(p, q, gq, begin, end, key, &s_n);
        uint64_t* out = p.parts + (int64_t)item * p.k;
        for (int j = threadIdx.x; j < p.k; j += SEL) out[j] = j < found ? key[j] : 0;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) s_last = atomicAdd(&p.done[t], 1) == splits - 1;
        __syncthreads();
        if (s_last) {
            __threadfence();
            if (threadIdx.x == 0) s_n = 0;
            __syncthreads();
            BestKeys<SEL> all = {key, &s_n, 0};
            const int64_t n = (int64_t)splits * p.k;
            const uint64_t* in = p.parts + (int64_t)(item - part) * p.k;
            for (int64_t r0 = 0; r0 < n; r0 += BestKeys<SEL>::BATCH) {
                for (int64_t i = r0 + threadIdx.x; i < r0 + BestKeys<SEL>::BATCH && i < n; i += SEL)
                    all.offer(__ldcg(in + i));
                found = all.settle(p.k, r0 + BestKeys<SEL>::BATCH >= n);
            }
            write_best<SEL>(p, t, key, found);
        }
        __syncthreads();
    }
}

static int round_up(int x, int a) { return (x + a - 1) / a * a; }

// Queries per tile.  A pair's time for a tile of rows is, per 64 elements, nt / 2 cycles of
// the tensor cores or, where that is more, the bytes that pass through each CTA's shared
// memory -- operands, the stage's copy, and the scale warps' reads -- at the 88 a cycle that
// fit what was measured (1M x 1536, us a tile: NV nt 128 1.77, 192 2.00, 256 2.40; MX 1.75,
// 1.83, 2.35); about 450 cycles more where one accumulator buffer has to be drained before
// the next tile.  Taken is the nt whose query tiles, spread over the pairs, take the least:
// 256 for a batch of 1024 (main pass NV 549 us against 727 at 192 and 834 at 128, MX 525, 640
// and 762), 16 for one query.
static bool search_plan(int fmt, int dp, int nq, int64_t n_tiles, Plan* out) {
    const int aps = atoms_per_stage(fmt), steps = dp / 64;
    const int kchunks = (dp / 2 + KC - 1) / KC;
    const int stage = A_BYTES + aps * 512;
    const int fixed = 1024 + 2 * MAX_NT * 4 + EPI_WARPS * HITS * 9 + (4 * MAX_STAGES + 9) * 8 + 64;
    constexpr int64_t pairs = 74;  // of the B200's 148 SMs
    double best = 0.0;
    bool any = false;
    for (int nt = 16; nt <= MAX_NT; nt += 16) {
        Plan s;
        s.nt = nt;
        s.nt_pad = round_up(nt, 128);
        s.kchunks = kchunks;
        s.n_qt = (nq + nt - 1) / nt;
        const int sf_tiles = s.nt_pad / 128, set = aps * 4;
        // an odd number of 16 columns is read with 16 more
        const int cols = (int)TMEM_COLS - (nt % 32 ? 16 : 0);
        const int sfb = kchunks * aps * 4 * sf_tiles;
        s.resident = nt + sfb + 2 * set <= cols;
        const int set_cols = s.resident ? set : set * (1 + sf_tiles);
        const int left = cols - (s.resident ? sfb : 0);
        if (nt + 2 * set_cols > left) continue;
        s.bufs = 2 * nt + 2 * set_cols <= left ? 2 : 1;
        const int held = kchunks * (nt / 2) * KC;
        const int streamed = s.resident ? 0 : sf_tiles * kchunks * aps * 512;
        s.stages = (SMEM_MAX - fixed - held - streamed) / stage;
        // the queries' scales pass through the ring
        if (s.stages < 3 || (s.resident && s.stages * stage < sf_tiles * kchunks * aps * 512)) continue;
        if (s.stages > MAX_STAGES) s.stages = MAX_STAGES;
        s.sets = (left - s.bufs * nt) / set_cols;
        if (s.sets > s.stages) s.sets = s.stages;
        s.smem = fixed + held + streamed + s.stages * stage;
        const double bytes = HALF * 32 + nt / 2 * 32 + stage / 4.0 + 4.0 * aps * 512 / 4 +
                             (s.resident ? 0.0 : 4.0 * aps * sf_tiles * 512 / 4);
        const double tensor = nt / 2.0;
        const double cycles = steps * (tensor > bytes / 88 ? tensor : bytes / 88) +
                              (s.bufs == 1 ? 450.0 : 0.0);
        const int64_t per = pairs / s.n_qt > 0 ? pairs / s.n_qt : 1;
        const int64_t waves = (s.n_qt * per + pairs - 1) / pairs;
        const double time = cycles * (double)((n_tiles + per - 1) / per) * (double)waves;
        if (!any || time < best * 0.999) {
            best = time;
            *out = s;
            any = true;
        }
    }
    return any;
}

// A call asks for the same plan several times: for its workspace, its queries and each launch.
static bool make_plan(int fmt, int dp, int nq, int64_t n_tiles, Plan* out) {
    thread_local int64_t of[4] = {-1, 0, 0, 0};
    thread_local Plan plan;
    thread_local bool ok = false;
    if (of[0] != fmt || of[1] != dp || of[2] != nq || of[3] != n_tiles) {
        ok = search_plan(fmt, dp, nq, n_tiles, &plan);
        of[0] = fmt;
        of[1] = dp;
        of[2] = nq;
        of[3] = n_tiles;
    }
    *out = plan;
    return ok;
}

}  // namespace fp4

int fp4_max_dim() { return fp4::kMaxDim; }
int fp4_cap() { return fp4::CAP; }
int fp4_tile_rows() { return fp4::ROWS; }

bool fp4_plan(int format, int dp, int nq, int64_t n_rows, Fp4Plan* out) {
    fp4::Plan s;
    if (!fp4::make_plan(format, dp, nq, (n_rows + fp4::ROWS - 1) / fp4::ROWS, &s)) return false;
    out->nt = s.nt;
    out->nt_pad = s.nt_pad;
    out->n_qt = s.n_qt;
    return true;
}

int launch_fp4_product(const Fp4Product& L, cudaStream_t st) {
    using namespace fp4;
    Plan s;
    const int dp = pad_dim(L.dim);
    const int64_t row_tiles = (L.n_rows + ROWS - 1) / ROWS;
    // the plan of the whole call, whatever part of the rows this launch takes: the queries
    // are laid out for it
    if (!make_plan(L.format, dp, L.nq, row_tiles, &s)) return PION_B200_ESHAPE;
    const int atoms = atoms_of(L.format, dp), aps = atoms_per_stage(L.format);
    const int64_t store_tiles = (L.store_rows + 127) / 128;
    CUtensorMap rows, row_sf, q, q_sf;
    if (make_tmap_2d(&rows, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, L.codes, (uint64_t)dp / 2,
                     (uint64_t)L.store_rows, (uint64_t)dp / 2, KC, HALF,
                     CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
        make_tmap_2d(&row_sf, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, L.scales, 128,
                     (uint64_t)store_tiles * atoms, 512, 128, (uint32_t)aps,
                     CU_TENSOR_MAP_SWIZZLE_NONE) != 0 ||
        make_tmap_2d(&q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, L.q_codes, (uint64_t)dp / 2,
                     (uint64_t)s.n_qt * s.nt_pad, (uint64_t)dp / 2, KC, (uint32_t)s.nt / 2,
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
    p.plan = s;
    p.mmas = dp / 64;
    p.atoms = atoms;
    p.n_tiles = L.n_tiles > 0 ? L.n_tiles : (int)row_tiles;
    p.tile_step = L.tile_step;
    p.tile_skip = L.tile_skip;
    p.out = L.out;
    p.out_type = L.out_type;
    p.ld = L.ld;
    p.theta = L.theta;
    p.cand_n = L.cand_n;
    p.cand = L.cand;
    p.status = L.status;
    p.wait_ns = L.wait_ns;
    p.test_stall = L.test_stall;
    // Pairs per query tile: one wave where there are enough SMs.  The query tiles of one row
    // tile run beside each other, so that the rows come from HBM once.
    int64_t per = L.num_sms / 2 / s.n_qt;
    if (per < 1) per = 1;
    if (per > p.n_tiles) per = p.n_tiles;
    const dim3 grid((unsigned)(2 * per * s.n_qt));
    const int mode = L.theta ? kCollect : kScores;
    const bool mx = L.format == kMX;
    const void* fn = mx ? (const void*)fp4_tc_kernel<kMX> : (const void*)fp4_tc_kernel<kNV>;
    if (set_smem_limit(fn, s.smem) != 0) return PION_B200_ECUDA;
    return mx ? launch_pdl(fp4_tc_kernel<kMX>, grid, THREADS, s.smem, st, rows, row_sf, q, q_sf, p, mode)
              : launch_pdl(fp4_tc_kernel<kNV>, grid, THREADS, s.smem, st, rows, row_sf, q, q_sf, p, mode);
}

int fp4_sample_tiles(int nq) { return nq <= 64 ? 64 : 32; }

int launch_fp4_theta(const float* sample, const uint64_t* cand, int k, int dim,
                     const float* q_scale, int nt, int nt_pad, const float* q_norm,
                     const float* norm_max, int nq, float* theta, int* cand_n, cudaStream_t st) {
    using namespace fp4;
    const int dp = pad_dim(dim);
    if (cand)
        return launch_pdl(theta_kernel, dim3((unsigned)nq), SEL, 0, st, cand, k, dp, q_scale, nt,
                          nt_pad, q_norm, norm_max, theta, cand_n);
    if (fp4_sample_tiles(nq) == 64) {
        static_assert(64 * ROWS == 1024 * 4 * 4, "sample");
        return launch_pdl(theta_sample_kernel<1024, 4>, dim3((unsigned)nq), 1024, 0, st, sample, k, dp,
                          q_scale, nt, nt_pad, q_norm, norm_max, theta, cand_n);
    }
    static_assert(32 * ROWS == 256 * 8 * 4, "sample");
    return launch_pdl(theta_sample_kernel<256, 8>, dim3((unsigned)nq), 256, 0, st, sample, k, dp,
                      q_scale, nt, nt_pad, q_norm, norm_max, theta, cand_n);
}

// Whether the scores of every row are written and split (they and the second pass over them
// cost less than a sample's own launch and selection), and the chunks' candidates fit.
bool fp4_splits(int64_t nq, int64_t n_rows, int64_t k) {
    const int64_t chunks = (n_rows + fp4::SPLIT - 1) / fp4::SPLIT;
    return chunks > 2 && nq * n_rows <= (int64_t)1 << 22 && chunks * k <= fp4::CAP / 2;
}

int launch_fp4_split(const float* scores, int64_t ld, int64_t n_rows, int k, int dim,
                     const float* q_scale, int nt, int nt_pad, const float* q_norm,
                     const float* norm_max, int nq, uint64_t* cand, int* cand_n, cudaStream_t st) {
    using namespace fp4;
    const dim3 grid((unsigned)((n_rows + SPLIT - 1) / SPLIT), (unsigned)nq);
    return launch_pdl(split_kernel, grid, SEL, 0, st, scores, ld, n_rows, k, pad_dim(dim), q_scale,
                      nt, nt_pad, q_norm, norm_max, cand, cand_n);
}

int64_t fp4_rescue_items(int64_t nq) { return nq > fp4::RESCUE_CTAS ? nq : fp4::RESCUE_CTAS; }

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
    p.nq = L.nq;
    p.n_flagged = L.n_flagged;
    p.flagged = L.flagged;
    p.done = L.done;
    p.parts = L.parts;
    const int smem = p.dp + p.dp / block_of(L.format) * 4;
    const dim3 grid((unsigned)L.nq);
    // Few queries: a CTA of 32 warps each, so that the dozen rows scored exactly are one round.
    const bool mx = L.format == kMX, few = L.nq <= 148;
    int rc;
    if (few)
        rc = mx ? launch_pdl(finish_kernel<kMX, 1024>, grid, 1024, smem, st, p)
                : launch_pdl(finish_kernel<kNV, 1024>, grid, 1024, smem, st, p);
    else
        rc = mx ? launch_pdl(finish_kernel<kMX, SEL>, grid, SEL, smem, st, p)
                : launch_pdl(finish_kernel<kNV, SEL>, grid, SEL, smem, st, p);
    if (rc != 0 || L.dense) return rc;
    return mx ? launch_pdl(rescue_kernel<kMX>, dim3(RESCUE_CTAS), SEL, smem, st, p)
              : launch_pdl(rescue_kernel<kNV>, dim3(RESCUE_CTAS), SEL, smem, st, p);
}

}  // namespace pion
