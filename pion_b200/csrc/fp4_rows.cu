// Microscaled 4-bit rows on B200: quantising rows as they are written into a store, and
// reading them back.  No counterpart in the reference, whose block formats are quantised on
// the host when an index is compacted (src/vector/kernels.mojo:1116-1842).
//
//   MX  block of 32: s = 2^(floor(log2 bmax) - 2), g = 1;  code = e2m1(x / s)
//   NV  block of 16: g = amax / 2688, s = e4m3(bmax / f32(6 g)), code = e2m1(x / f32(s g))
//   read: x = f32((code s) g), then rounded to the output type
//
// Every quotient is rounded once, as the exact quotient would be: a fast path multiplies by
// the reciprocal and converts the product's two neighbours 2^-21 away; where they agree no
// value in between (the exact quotient among them) rounds elsewhere, and where they do not the
// borders are compared exactly.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "fp4.cuh"
#include "internal.h"

namespace pion {
namespace fp4 {

constexpr int WARPS = 8;   // per CTA that writes one row
constexpr int NW = 2;      // per CTA that writes several: its place is soon free for the next
                           // (262144 x 1536 float32, us with 8 and with 2: NV 344 and 321, MX 304
                           // and 292)
constexpr int READ_WARPS = 4;  // (262144 x 1536 bfloat16, us with 8 and with 4: 170 and 166)
constexpr int FEW = 1024;  // rows written by a CTA each
constexpr int STEP = 256;  // elements per warp step, eight consecutive ones per lane

// In NV an amax below this is stored as a row of zeros: g = amax / 2688 and its multiples then stay
// normal numbers.
__device__ constexpr float kTiny = 0x1p-100f;

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// The larger magnitude, NaN if either is.
__device__ __forceinline__ float max_abs(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)));
    return m;
}

// Eight consecutive elements as they are in memory, their values and their largest magnitude
// (NaN if one is).
template <class T>
struct alignas(16) Eight {
    T x[8];
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
                v[2 * j] = (float)x[2 * j];
                v[2 * j + 1] = (float)x[2 * j + 1];
            } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(w + j));
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ float top() const {
        if constexpr (sizeof(T) == 4) {
            return max_abs(max_abs(max_abs(x[0], x[1]), max_abs(x[2], x[3])),
                           max_abs(max_abs(x[4], x[5]), max_abs(x[6], x[7])));
        } else {  // two at a time; a NaN stays one
            const uint4 w = *reinterpret_cast<const uint4*>(x);
            const uint32_t m = 0x7FFF7FFFu;
            uint32_t a = max16(w.x & m, w.y & m), b = max16(w.z & m, w.w & m);
            a = max16(a, b);
            a = max16(a, a >> 16) & 0xFFFFu;
            if constexpr (std::is_same<T, __nv_bfloat16>::value)
                return __uint_as_float(a << 16);
            else
                return __half2float(__ushort_as_half((unsigned short)a));
        }
    }
    // magnitudes order as integers, infinity and then NaN above all
    static __device__ __forceinline__ uint32_t max16(uint32_t a, uint32_t b) {
        return __vmaxu2(a, b);
    }
};

// The eight elements from column c0 + 8 * lane of a row, zeros past dim.  VEC: rows start at
// 16-byte boundaries; else the warp's 256 elements come in one by one, side by side, and pass
// through shared memory.  FULL: all of them lie inside the row.
template <class T, bool VEC, bool FULL = false>
__device__ __forceinline__ Eight<T> load8(const T* row, int c0, int dim, int lane, T* stage) {
    const int c = c0 + 8 * lane;
    Eight<T> e;
    if constexpr (VEC) {
        if (FULL || c + 8 <= dim) {
            constexpr int N = sizeof(Eight<T>) / 16;
            uint4* raw = reinterpret_cast<uint4*>(&e);
#pragma unroll
            for (int j = 0; j < N; ++j) raw[j] = __ldcg(reinterpret_cast<const uint4*>(row + c) + j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) e.x[j] = c + j < dim ? __ldcg(row + c + j) : from_float<T>(0.0f);
        }
    } else {
        T x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int at = c0 + 32 * j + lane;
            x[j] = FULL || at < dim ? __ldcg(row + at) : from_float<T>(0.0f);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) stage[32 * j + lane] = x[j];
        __syncwarp();
        e = *reinterpret_cast<const Eight<T>*>(stage + 8 * lane);
    }
    return e;
}

__device__ __forceinline__ float rcp_approx(float x) {  // within an ulp, x normal
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// The e4m3 byte nearest to top / h (top >= 0, h > 0, quotient at most 448 (1 + 2^-22)); rh is
// 1 / h within 2^-22.
__device__ __forceinline__ uint32_t e4m3_quotient(float top, float h, float rh) {
    const float t = top * rh;
    uint32_t two;  // the neighbours' bytes, the lower one first
    asm("{\n\t.reg .b16 t;\n\tcvt.rn.satfinite.e4m3x2.f32 t, %2, %1;\n\tcvt.u32.u16 %0, t;\n\t}"
        : "=r"(two)
        : "f"(t * (1.0f - 0x1p-20f)), "f"(t * (1.0f + 0x1p-20f)));
    const uint32_t lo = two & 0xFFu, hi = two >> 8;
    if (lo == hi) return lo;
    // the neighbours' border has five significant bits: the fused multiply-add's sign is that
    // of the exact top - border h
    const float over = fmaf(-0.5f * (e4m3_value(lo) + e4m3_value(hi)), h, top);
    return over > 0.0f || (over == 0.0f && (lo & 1u)) ? hi : lo;
}

// Where the codes of a value's two neighbours differ, the one that is nearest to v / d: the
// border between two codes c and c + 1 has three significant bits, so the fused multiply-add's
// sign is that of the exact |v| - border d.  `lo` holds the codes nearer to zero.
__device__ __forceinline__ uint32_t settle_borders(uint32_t lo, uint32_t hi, const float (&v)[8],
                                                   float d) {
    uint32_t open = lo ^ hi;
    while (open) {
        const int j = (__ffs(open) - 1) >> 2;
        float x = v[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) x = j == i ? v[i] : x;
        const uint32_t c = (lo >> (4 * j)) & 7u;
        const float border = c < 4 ? 0.25f + 0.5f * (float)c : c == 4 ? 2.5f : c == 5 ? 3.5f : 5.0f;
        const float over = fmaf(-border, d, fabsf(x));
        if (over > 0.0f || (over == 0.0f && (c & 1u))) lo += 1u << (4 * j);
        open &= ~(15u << (4 * j));
    }
    return lo;
}

// v r, two products an instruction.
__device__ __forceinline__ void mul8(float (&out)[8], const float (&v)[8], float r) {
#pragma unroll
    for (int j = 0; j < 8; j += 2)
        asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\t"
            "mul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
            : "=f"(out[j]), "=f"(out[j + 1])
            : "f"(v[j]), "f"(v[j + 1]), "f"(r));
}

// Eight codes of v / d; rd is 1 / d, in MX exactly, in NV within 2^-22 (0 for d = 0).
template <int FMT>
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float d, float rd) {
    float a[8];
    if (FMT == kMX) {  // a power of two: the product is the quotient
        mul8(a, v, rd);
        return e2m1x8(a);
    }
    float b[8];
    mul8(a, v, rd * (1.0f - 0x1p-21f));
    mul8(b, v, rd * (1.0f + 0x1p-21f));
    const uint32_t lo = e2m1x8(a), hi = e2m1x8(b);
    return lo == hi ? lo : settle_borders(lo, hi, v, d);
}

struct WriteParams {
    const void* src;
    int64_t stride;        // elements between rows
    int64_t n;
    const int64_t* slots;  // null: row i goes to slot start + i
    int64_t start;
    int64_t n_slots;
    int32_t* claim;        // with slots: the last row of a slot's rows, plus one
    int tile, tile_pad;    // > 0: a query batch, slot = query_slot(i)
    int dim, dp;
    uint8_t* codes;
    uint8_t* scales;
    float* row_scale;
    float* norm;           // per row (queries), or null
    float* norm_max;       // the store's bound, or null
    int* zero;             // n + 1 integers set to 0, or null
    int* status;
};

// A slot named by several rows of one write keeps the last of them.  Of few rows each CTA looks
// through the rows after its own; of many, every row first raises the slot's claim to its
// index, and the write kernel takes only the row that holds it.
__global__ void claim_kernel(const int64_t* slots, int64_t n, int64_t n_slots,
                             int32_t* claim, int* status) {
    griddep_launch();
    griddep_wait();
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int64_t s = __ldcg(slots + i);
    if (s >= n_slots) record_error(status, PION_B200_EINVAL);
    if (s >= 0 && s < n_slots) atomicMax(&claim[s], (int32_t)(i + 1));
}

// A barrier of the row's warps, `base` the first of them.
template <int WPR>
__device__ __forceinline__ void row_sync(int base) {
    asm volatile("bar.sync %0, %1;" ::"r"(1 + base / WPR), "n"(WPR * 32) : "memory");
}

// WPR warps per row: one or two where rows are many, the CTA's eight where they are few and a
// row's own latency counts.  An MX row is one pass.  NV needs the row's largest magnitude first; its
// elements stay in registers between the two passes where a warp's share is at most HOLD
// steps (HOLD = 0: they are read again).  The first OPEN steps of a warp (in MX all, if any) lie
// inside the row and are not checked against its end.  Bound by HBM: the row, its codes, scales
// and g once.
template <int FMT, class T, bool VEC, int W, int WPR, int HOLD, int OPEN>
__global__ void __launch_bounds__(W * 32) write_kernel(const WriteParams p) {
    __shared__ __align__(16) T stage_all[VEC ? 1 : W * STEP];
    __shared__ float s_max[W];
    __shared__ float s_s2[W];
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T* stage = stage_all + (VEC ? 0 : warp * STEP);
    const int64_t i = (int64_t)blockIdx.x * (W / WPR) + warp / WPR;
    const int mine = warp % WPR;               // of the row's warps
    const int base = warp - mine;
    if (i >= p.n) return;
    if (p.zero && lane == 0 && mine == 0) {
        p.zero[i + 1] = 0;
        if (i == 0) p.zero[0] = 0;
    }
    int64_t slot;
    if (p.tile > 0) {
        slot = query_slot(i, p.tile, p.tile_pad);
    } else if (p.slots) {
        slot = __ldcg(p.slots + i);
        if (WPR == WARPS) {
            bool later = false;
            for (int64_t j = i + 1 + threadIdx.x; j < p.n; j += WARPS * 32)
                later |= __ldcg(p.slots + j) == slot;
            if (__syncthreads_or(later)) return;
            if (slot >= p.n_slots && threadIdx.x == 0) record_error(p.status, PION_B200_EINVAL);
        }
        if (slot < 0 || slot >= p.n_slots) return;
        if (WPR < WARPS && __ldcg(p.claim + slot) != (int32_t)(i + 1)) return;
    } else {
        slot = p.start + i;
    }
    const T* row = static_cast<const T*>(p.src) + i * p.stride;
    const int atoms = atoms_of(FMT, p.dp);
    constexpr int BL = block_of(FMT) / 8;  // lanes per block
    const int steps = (p.dp + STEP - 1) / STEP;
    const int first = mine;
    uint32_t* codes_out = reinterpret_cast<uint32_t*>(p.codes + slot * (p.dp / 2)) + lane;
    uint8_t* scales_out = p.scales + scale_word(slot, lane / (4 * BL), atoms);

    float amax = 0.0f;  // of this warp's elements, then of the row: NaN and infinities show
    float s2 = 0.0f;    // sum of the blocks' squared scales, BL times over
    float g = 1.0f, h = 1.0f, rh = 1.0f;
    bool live = true;
    auto row_max = [&]() {
#pragma unroll
        for (int o = 16; o; o >>= 1) amax = max_abs(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if constexpr (WPR > 1) {
            if (lane == 0) s_max[warp] = amax;
            row_sync<WPR>(base);
#pragma unroll
            for (int w = 0; w < WPR; ++w) amax = max_abs(amax, s_max[base + w]);
        }
    };
    auto quantise = [&](int k, const float(&v)[8], float top, bool open) {
        const int c = k * STEP + lane * 8;
#pragma unroll
        for (int o = 1; o < BL; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        uint32_t bits = 0, codes = 0;
        if (FMT == kMX) {
            // floor(log2 top) - 2 as a biased exponent, at least the format's least (at most
            // 252, infinities aside)
            const int e = (int)(__float_as_uint(top) >> 23) - 2;
            bits = (uint32_t)min(max(e, 0), 252);
            const float d = e8m0_value(bits);
            s2 = fmaf(d, d, s2);
            codes = codes8<FMT>(v, d, __uint_as_float((254u - bits) << 23));  // 2^(127 - bits)
        } else if (live) {
            bits = e4m3_quotient(top, h, rh);
            const float s = e4m3_value(bits);
            const float d = __fmul_rn(s, g);
            s2 = fmaf(s, s, s2);
            codes = codes8<FMT>(v, d, bits ? rcp_approx(d) : 0.0f);
        }
        if (open || c < p.dp) codes_out[k * 32] = codes;
        // four blocks' bytes to the first lane of their atom
        uint32_t word = bits << (8 * ((lane / BL) & 3));
#pragma unroll
        for (int o = BL; o < 4 * BL; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
        if ((open || c < p.dp) && lane % (4 * BL) == 0)
            *reinterpret_cast<uint32_t*>(scales_out + k * (STEP / (32 * BL)) * 512) = word;
    };
    if constexpr (FMT == kMX) {
        // four steps' loads in flight
        for (int k0 = first; k0 < steps; k0 += 4 * WPR) {
            Eight<T> e[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k0 + u * WPR < steps)
                    e[u] = load8<T, VEC, (OPEN > 0)>(row, (k0 + u * WPR) * STEP, p.dim, lane, stage);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (k0 + u * WPR < steps) {
                    float v[8];
                    e[u].values(v);
                    const float top = e[u].top();
                    amax = max_abs(amax, top);
                    quantise(k0 + u * WPR, v, top, OPEN > 0);
                }
        }
        row_max();
        if (amax == 0.0f) g = 0.0f;
    } else {
        constexpr int H = HOLD > 0 ? HOLD : 1;
        Eight<T> e[H];
        float v[8], top[H];
        if constexpr (HOLD > 0) {
#pragma unroll
            for (int u = 0; u < H; ++u)
                if (u < OPEN)
                    e[u] = load8<T, VEC, true>(row, (first + u * WPR) * STEP, p.dim, lane, stage);
                else if (first + u * WPR < steps)
                    e[u] = load8<T, VEC>(row, (first + u * WPR) * STEP, p.dim, lane, stage);
#pragma unroll
            for (int u = 0; u < H; ++u)
                if (u < OPEN || first + u * WPR < steps) amax = max_abs(amax, top[u] = e[u].top());
        } else {
            for (int k = first; k < steps; k += WPR) {
                amax = max_abs(amax, load8<T, VEC>(row, k * STEP, p.dim, lane, stage).top());
            }
        }
        row_max();
        live = amax >= kTiny && amax < INFINITY;
        g = live ? __fdiv_rn(amax, 2688.0f) : 0.0f;
        h = live ? __fmul_rn(6.0f, g) : 1.0f;
        rh = rcp_approx(h);
        if constexpr (HOLD > 0) {
#pragma unroll
            for (int u = 0; u < H; ++u)
                if (u < OPEN || first + u * WPR < steps) {
                    e[u].values(v);
                    quantise(first + u * WPR, v, top[u], u < OPEN);
                }
        } else {
            for (int k = first; k < steps; k += WPR) {
                e[0] = load8<T, VEC>(row, k * STEP, p.dim, lane, stage);
                e[0].values(v);
                quantise(k, v, e[0].top(), false);
            }
        }
    }
    const bool fine = amax < INFINITY;
#pragma unroll
    for (int o = 16; o; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    if constexpr (WPR > 1) {
        if (lane == 0) s_s2[warp] = s2;
        row_sync<WPR>(base);
        if (mine != 0) return;
        s2 = 0.0f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) s2 += s_s2[base + w];
    }
    if (lane == 0) {
        p.row_scale[slot] = fine ? g : __int_as_float(0x7fc00000);
        // every element is at most 6 s g: |row| <= 6 g sqrt(block * sum s^2); where the squares
        // of MX scales could leave the normal numbers, no element is more than twice amax
        float bound = 6.02f * g * sqrtf((float)(block_of(FMT) / BL) * s2);
        if (FMT == kMX && !(s2 >= 0x1p-100f && s2 < 0x1p100f))
            bound = 2.01f * amax * sqrtf((float)p.dim);
        if (!fine) bound = 0.0f;
        if (p.norm) p.norm[i] = bound;
        if (p.norm_max && bound > __ldcg(p.norm_max))
            atomicMax(reinterpret_cast<int*>(p.norm_max), __float_as_int(bound));
        if (WPR < WARPS && p.slots) p.claim[slot] = 0;
    }
}

struct ReadParams {
    const uint8_t* codes;
    const uint8_t* scales;
    const float* row_scale;
    int64_t n_slots;
    const int64_t* slots;  // null: start + i
    int64_t start;
    int64_t n;
    int dim, dp;
    void* dst;
    int64_t stride;
    int* status;
};

__device__ __forceinline__ void store8(float* to, const float (&t)[8]) {  // a whole sector a lane
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "f"(t[0]),
                 "f"(t[1]), "f"(t[2]), "f"(t[3]), "f"(t[4]), "f"(t[5]), "f"(t[6]), "f"(t[7])
                 : "memory");
}
template <class T>
__device__ __forceinline__ void store8(T* to, const T (&t)[8]) {
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(t);
}

// One warp per row.  Bound by HBM: the output once.
template <int FMT, class T, bool VEC>
__global__ void __launch_bounds__(READ_WARPS * 32) read_kernel(const ReadParams p) {
    __shared__ __align__(16) T stage_all[VEC ? 1 : READ_WARPS * STEP];
    griddep_launch();
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T* stage = stage_all + (VEC ? 0 : warp * STEP);
    const int64_t i = (int64_t)blockIdx.x * READ_WARPS + warp;
    if (i >= p.n) return;
    const int64_t slot = p.slots ? __ldcg(p.slots + i) : p.start + i;
    if (slot < 0) return;
    if (slot >= p.n_slots) {
        if (lane == 0) record_error(p.status, PION_B200_EINVAL);
        return;
    }
    const float g = __ldcg(&p.row_scale[slot]);
    const int atoms = atoms_of(FMT, p.dp);
    constexpr int BL = block_of(FMT) / 8;              // lanes per block
    constexpr int APB = 8 * STEP / (4 * block_of(FMT));  // atoms of eight steps, at most a warp's
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.codes + slot * (p.dp / 2)) + lane;
    const uint8_t* scales = p.scales + scale_word(slot, 0, atoms);
    T* out = static_cast<T*>(p.dst) + i * p.stride;
    // Eight steps' loads in flight: a word of codes a lane and step, and the scale bytes of an
    // atom a lane, handed round by shuffles.
    for (int c00 = 0; c00 < p.dim; c00 += 8 * STEP) {
        const int atom0 = c00 / (4 * block_of(FMT));
        const uint32_t bytes = lane < APB && atom0 + lane < atoms
                                   ? __ldcg(reinterpret_cast<const uint32_t*>(
                                         scales + (int64_t)(atom0 + lane) * 512))
                                   : 0u;
        uint32_t packed[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            packed[u] = c00 + u * STEP + 8 * lane < p.dp ? __ldcg(codes + c00 / 8 + u * 32) : 0u;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int c0 = c00 + u * STEP;
            if (c0 >= p.dim) break;
            const int c = c0 + 8 * lane;
            const uint32_t word =
                __shfl_sync(0xffffffffu, bytes, u * (STEP / (4 * block_of(FMT))) + lane / (4 * BL));
            const float s = scale_value<FMT>((word >> (8 * ((lane / BL) & 3))) & 255u);
            float v[8];
            e2m1x8_values(packed[u], v);
            // code * s has at most six significant bits: one rounding in the product with g
            // (and one to a 16-bit output, from a value already within 2^-24)
            alignas(16) T t[8];
            mul8(v, v, s);
            mul8(v, v, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = from_float<T>(v[j]);
            if constexpr (VEC) {
                if (c + 8 <= p.dim) {
                    store8(out + c, t);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (c + j < p.dim) out[c + j] = t[j];
                }
            } else {
                // side by side through shared memory: eight strided elements a lane took more
                // than twice as long
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) stage[8 * lane + j] = t[j];
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = 32 * j + lane;
                    if (c0 + e < p.dim) out[c0 + e] = stage[e];
                }
            }
        }
    }
}

template <int FMT, class T, bool VEC, int WPR, int HOLD, int OPEN>
static int write_many(const WriteParams& p, cudaStream_t st) {
    constexpr int ROWS = NW / WPR;
    return launch_pdl(write_kernel<FMT, T, VEC, NW, WPR, HOLD, OPEN>,
                      dim3((unsigned)((p.n + ROWS - 1) / ROWS)), NW * 32, 0, st, p);
}

// NV rows that fill WPR warps' HOLD steps, all but the last, and others.
template <class T, bool VEC, int WPR, int HOLD>
static int write_held(const WriteParams& p, cudaStream_t st) {
    if (p.dim == WPR * HOLD * STEP) return write_many<kNV, T, VEC, WPR, HOLD, HOLD>(p, st);
    if (p.dim >= WPR * (HOLD - 1) * STEP) return write_many<kNV, T, VEC, WPR, HOLD, HOLD - 1>(p, st);
    return write_many<kNV, T, VEC, WPR, HOLD, 0>(p, st);
}

template <int FMT, class T, bool VEC>
static int write_v(const WriteParams& p, cudaStream_t st) {
    // Few rows: a CTA each; many: a warp each (NV float32, 1536 elements, us a write in a graph of
    // them: 148 rows 2.3 and 2.6, 1024 rows 4.7 and 4.7, 2048 rows 8.2 and 5.1).
    if (p.n <= FEW)
        return launch_pdl(write_kernel<FMT, T, VEC, WARPS, WARPS, 4, 0>, dim3((unsigned)p.n),
                          WARPS * 32, 0, st, p);
    if constexpr (FMT == kNV) {
        // A row stays in one warp's registers while that leaves room for enough warps, else in two
        // warps', and is read twice only where neither holds it.  Steps known to lie inside the row
        // are not checked against its end.  Medians of writes in turn, us:
        //                            one warp   two warps   read twice   the variant taken, checked
        //   262144 x 1536  float32      321         330         431          349
        //                  bfloat16     225         278         395          270
        //   131072 x 2048  float32      247         222         296          243
        //                  bfloat16     148         173         262          181
        //   65536 x 4096   float32                  244         307          280
        //                  bfloat16                 161         259          196
        //   100000 x 777   float16       67                                   76
        //   60000 x 1900   float16       76                                   90
        if (p.dp <= 3 * STEP) return write_held<T, VEC, 1, 3>(p, st);
        if (p.dp <= 4 * STEP) return write_held<T, VEC, 1, 4>(p, st);
        if (p.dp <= 6 * STEP) return write_held<T, VEC, 1, 6>(p, st);
        if (p.dp <= 8 * STEP) {
            if constexpr (sizeof(T) == 4)
                return write_held<T, VEC, 2, 4>(p, st);
            else
                return write_held<T, VEC, 1, 8>(p, st);
        }
        if (p.dp <= 16 * STEP) return write_held<T, VEC, 2, 8>(p, st);
        return write_many<FMT, T, VEC, 1, 0, 0>(p, st);
    } else {
        return p.dim % STEP == 0 ? write_many<FMT, T, VEC, 1, 0, 1>(p, st)
                                 : write_many<FMT, T, VEC, 1, 0, 0>(p, st);
    }
}

template <int FMT, class T>
static int write_t(const WriteParams& p, cudaStream_t st) {
    static_assert(kMaxDim <= WARPS * 4 * STEP, "a CTA holds a row");
    const bool vec = reinterpret_cast<uintptr_t>(p.src) % 16 == 0 && p.stride * sizeof(T) % 16 == 0;
    return vec ? write_v<FMT, T, true>(p, st) : write_v<FMT, T, false>(p, st);
}

template <int FMT, class T>
static int read_t(const ReadParams& p, cudaStream_t st) {
    constexpr size_t A = 8 * sizeof(T);
    const bool vec = reinterpret_cast<uintptr_t>(p.dst) % A == 0 && p.stride * sizeof(T) % A == 0;
    const dim3 grid((unsigned)((p.n + READ_WARPS - 1) / READ_WARPS));
    return vec ? launch_pdl(read_kernel<FMT, T, true>, grid, READ_WARPS * 32, 0, st, p)
               : launch_pdl(read_kernel<FMT, T, false>, grid, READ_WARPS * 32, 0, st, p);
}

}  // namespace fp4

int fp4_write_launches(bool slots, int64_t n) { return slots && n > fp4::FEW ? 2 : 1; }

int launch_fp4_write(const Fp4Write& w, cudaStream_t st) {
    using namespace fp4;
    if (w.n <= 0) return 0;
    if (fp4_write_launches(w.slots != nullptr, w.n) > 1) {
        if (launch_pdl(claim_kernel, dim3((unsigned)((w.n + 255) / 256)), 256, 0, st, w.slots, w.n,
                       w.n_slots, w.claim, w.status) != 0)
            return PION_B200_ECUDA;
    }
    WriteParams p;
    p.src = w.src;
    p.stride = w.stride;
    p.n = w.n;
    p.slots = w.slots;
    p.start = w.start;
    p.n_slots = w.n_slots;
    p.claim = w.claim;
    p.tile = w.tile;
    p.tile_pad = w.tile_pad;
    p.dim = w.dim;
    p.dp = pad_dim(w.dim);
    p.codes = w.codes;
    p.scales = w.scales;
    p.row_scale = w.row_scale;
    p.norm = w.norm;
    p.norm_max = w.norm_max;
    p.zero = w.zero;
    p.status = w.status;
    const bool mx = w.format == kMX;
    switch (w.type) {
        case PION_B200_F32: return mx ? write_t<kMX, float>(p, st) : write_t<kNV, float>(p, st);
        case PION_B200_BF16:
            return mx ? write_t<kMX, __nv_bfloat16>(p, st) : write_t<kNV, __nv_bfloat16>(p, st);
        default: return mx ? write_t<kMX, __half>(p, st) : write_t<kNV, __half>(p, st);
    }
}

int launch_fp4_read(const Fp4Read& r, cudaStream_t st) {
    using namespace fp4;
    if (r.n <= 0) return 0;
    ReadParams p;
    p.codes = r.codes;
    p.scales = r.scales;
    p.row_scale = r.row_scale;
    p.n_slots = r.n_slots;
    p.slots = r.slots;
    p.start = r.start;
    p.n = r.n;
    p.dim = r.dim;
    p.dp = pad_dim(r.dim);
    p.dst = r.dst;
    p.stride = r.stride;
    p.status = r.status;
    const bool mx = r.format == kMX;
    switch (r.type) {
        case PION_B200_F32: return mx ? read_t<kMX, float>(p, st) : read_t<kNV, float>(p, st);
        case PION_B200_BF16:
            return mx ? read_t<kMX, __nv_bfloat16>(p, st) : read_t<kNV, __nv_bfloat16>(p, st);
        default: return mx ? read_t<kMX, __half>(p, st) : read_t<kNV, __half>(p, st);
    }
}

}  // namespace pion
