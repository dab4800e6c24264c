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

#include "fp4.cuh"
#include "internal.h"

namespace pion {
namespace fp4 {

constexpr int WARPS = 8;  // rows in flight per CTA, a warp each
constexpr int STEP = 256; // elements per warp step, eight consecutive ones per lane

// amax below this is stored as a row of zeros: g = amax / 2688 and its multiples then stay
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

// Eight consecutive elements from column c of a row, zeros past dim.  VEC: the row starts at
// a 16-byte boundary.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int c, int dim, float (&v)[8]) {
    if (VEC && c + 8 <= dim) {
        constexpr int N = 8 * sizeof(T) / 16;
        alignas(16) uint4 raw[N];
#pragma unroll
        for (int j = 0; j < N; ++j) raw[j] = __ldg(reinterpret_cast<const uint4*>(row + c) + j);
        const T* t = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float<T>(t[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < dim ? to_float<T>(row[c + j]) : 0.0f;
    }
}

__device__ __forceinline__ float max8(const float (&v)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
    return m;
}

// The e4m3 byte nearest to top / h (top >= 0, h > 0, quotient at most 448 (1 + 2^-22)).
__device__ __forceinline__ uint32_t e4m3_quotient(float top, float h) {
    const float t = __fdividef(top, h);
    const uint32_t lo = e4m3_byte(t * (1.0f - 0x1p-20f)), hi = e4m3_byte(t * (1.0f + 0x1p-20f));
    if (lo == hi) return lo;
    // neighbours: compare top with the exact border (5 significant bits) times h
    const double mid = 0.5 * ((double)e4m3_value(lo) + (double)e4m3_value(hi)) * (double)h;
    if ((double)top == mid) return (lo & 1u) ? hi : lo;
    return (double)top > mid ? hi : lo;
}

// The e2m1 code of |x| / d by the borders themselves; the fused multiply-add's sign is that
// of the exact x - border d.
__device__ __noinline__ uint32_t e2m1_exact(float x, float d) {
    const float a = fabsf(x);
    uint32_t c = 0;
    c += fmaf(-0.25f, d, a) > 0.0f;
    c += fmaf(-0.75f, d, a) >= 0.0f;
    c += fmaf(-1.25f, d, a) > 0.0f;
    c += fmaf(-1.75f, d, a) >= 0.0f;
    c += fmaf(-2.5f, d, a) > 0.0f;
    c += fmaf(-3.5f, d, a) >= 0.0f;
    c += fmaf(-5.0f, d, a) > 0.0f;
    return c | (x < 0.0f ? 8u : 0u);
}

// Eight codes of v / d; rd = 1 / d rounded (0 for d = 0).
template <int FMT>
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], float d, float rd) {
    float a[8];
    if (FMT == kMX) {  // a power of two: the product is the quotient
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = v[j] * rd;
        return e2m1x8(a);
    }
    float b[8];
    const float r0 = rd * (1.0f - 0x1p-21f), r1 = rd * (1.0f + 0x1p-21f);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        a[j] = v[j] * r0;
        b[j] = v[j] * r1;
    }
    const uint32_t lo = e2m1x8(a), hi = e2m1x8(b);
    if (lo == hi) return lo;
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) c |= e2m1_exact(v[j], d) << (4 * j);
    return c;
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
    int* status;
};

// A slot named by several rows of one write keeps the last of them: every row raises the
// slot's claim to its index, and the write kernel takes only the row that holds it.
__global__ void claim_kernel(const int64_t* __restrict__ slots, int64_t n, int64_t n_slots,
                             int32_t* claim, int* status) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n) return;
    const int64_t s = slots[i];
    if (s >= n_slots) record_error(status, PION_B200_EINVAL);
    if (s >= 0 && s < n_slots) atomicMax(&claim[s], (int32_t)(i + 1));
}

// One warp per row.  Bound by HBM: the row once (the NV format's second pass finds it in L1),
// its codes, scales and g once.
template <int FMT, class T, bool VEC>
__global__ void __launch_bounds__(WARPS * 32) write_kernel(WriteParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (i >= p.n) return;
    int64_t slot;
    if (p.tile > 0) {
        slot = query_slot(i, p.tile, p.tile_pad);
    } else if (p.slots) {
        slot = p.slots[i];
        if (slot < 0 || slot >= p.n_slots) return;
        if (*(volatile int32_t*)&p.claim[slot] != (int32_t)(i + 1)) return;
    } else {
        slot = p.start + i;
    }
    const T* row = static_cast<const T*>(p.src) + i * p.stride;
    const int atoms = atoms_of(FMT, p.dp);
    constexpr int BL = block_of(FMT) / 8;  // lanes per block

    float amax = 0.0f;
    bool fine = true;  // no NaN or infinity in the row
    for (int c = lane * 8; c < p.dp; c += STEP) {
        float v[8];
        load8<T, VEC>(row, c, p.dim, v);
        float z = 0.0f;  // 0 * NaN and 0 * inf are NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) z = fmaf(v[j], 0.0f, z);
        fine = fine && z == 0.0f;
        amax = fmaxf(amax, max8(v));
    }
    fine = __all_sync(0xffffffffu, fine);
#pragma unroll
    for (int o = 16; o; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    const bool live = fine && (FMT == kMX ? amax > 0.0f : amax >= kTiny);
    float g = 0.0f, h = 1.0f;
    if (live) {
        g = FMT == kMX ? 1.0f : __fdiv_rn(amax, 2688.0f);
        h = __fmul_rn(6.0f, g);
    }

    float s2 = 0.0f;  // sum of the blocks' squared scales
    const int steps = (p.dp + STEP - 1) / STEP;
    for (int k = 0; k < steps; ++k) {
        const int c = k * STEP + lane * 8;
        float v[8];
        load8<T, VEC>(row, c, p.dim, v);
        float top = max8(v);
#pragma unroll
        for (int o = 1; o < BL; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        uint32_t bits = 0, codes = 0;
        if (live) {
            float d, rd;
            if (FMT == kMX) {
                // floor(log2 top) - 2 as a biased exponent, at least the format's least
                const int e = (int)(__float_as_uint(top) >> 23) - 2;
                bits = (uint32_t)(e < 0 ? 0 : e);
                d = e8m0_value(bits);
                rd = __uint_as_float((254u - bits) << 23);  // 2^(127 - bits), bits <= 252
                s2 = fmaf(d, d, s2);
            } else {
                bits = e4m3_quotient(top, h);
                const float s = e4m3_value(bits);
                d = __fmul_rn(s, g);
                rd = bits ? __frcp_rn(d) : 0.0f;
                s2 = fmaf(s, s, s2);
            }
            codes = codes8<FMT>(v, d, rd);
        }
        if (c < p.dp)
            reinterpret_cast<uint32_t*>(p.codes + slot * (p.dp / 2))[c >> 3] = codes;
        // four blocks' bytes to the first lane of their atom
        uint32_t word = bits << (8 * ((lane / BL) & 3));
#pragma unroll
        for (int o = BL; o < 4 * BL; o <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
        if (c < p.dp && lane % (4 * BL) == 0)
            *reinterpret_cast<uint32_t*>(p.scales +
                                         scale_word(slot, c / (32 * BL), atoms)) = word;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s2 += __shfl_xor_sync(0xffffffffu, s2, o);
    if (lane == 0) {
        p.row_scale[slot] = fine ? g : __int_as_float(0x7fc00000);
        // every element is at most 6 s g: |row| <= 6 g sqrt(block * sum s^2).  Every lane of
        // a block added its scale, BL times in all.
        const float bound =
            fine ? 6.02f * g * sqrtf((float)(block_of(FMT) / BL) * s2) : 0.0f;
        if (p.norm) p.norm[i] = bound;
        if (p.norm_max && bound > *(volatile float*)p.norm_max)
            atomicMax(reinterpret_cast<int*>(p.norm_max), __float_as_int(bound));
        if (p.slots) p.claim[slot] = 0;
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

template <int FMT, class T, bool VEC>
__global__ void __launch_bounds__(WARPS * 32) read_kernel(ReadParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (i >= p.n) return;
    const int64_t slot = p.slots ? p.slots[i] : p.start + i;
    if (slot < 0) return;
    if (slot >= p.n_slots) {
        if (lane == 0) record_error(p.status, PION_B200_EINVAL);
        return;
    }
    const float g = __ldg(&p.row_scale[slot]);
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(p.codes + slot * (p.dp / 2));
    const int atoms = atoms_of(FMT, p.dp);
    T* out = static_cast<T*>(p.dst) + i * p.stride;
    for (int c = lane * 8; c < p.dim; c += STEP) {
        float v[8];
        e2m1x8_values(__ldg(codes + (c >> 3)), v);
        const int b = c / block_of(FMT);
        const float s = scale_value<FMT>(__ldg(p.scales + scale_word(slot, b >> 2, atoms) + (b & 3)));
        // code * s has at most six significant bits: one rounding in the product with g (and
        // one to a 16-bit output, from a value already within 2^-24)
        alignas(16) T t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = from_float<T>(__fmul_rn(__fmul_rn(v[j], s), g));
        if (VEC && c + 8 <= p.dim) {
            constexpr int N = 8 * sizeof(T) / 16;
#pragma unroll
            for (int j = 0; j < N; ++j)
                reinterpret_cast<uint4*>(out + c)[j] = reinterpret_cast<const uint4*>(t)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < p.dim) out[c + j] = t[j];
        }
    }
}

template <int FMT, class T>
static int write_t(const WriteParams& p, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(p.src) % 16 == 0 && p.stride * sizeof(T) % 16 == 0;
    const dim3 grid((unsigned)((p.n + WARPS - 1) / WARPS));
    if (vec)
        write_kernel<FMT, T, true><<<grid, WARPS * 32, 0, st>>>(p);
    else
        write_kernel<FMT, T, false><<<grid, WARPS * 32, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : PION_B200_ECUDA;
}

template <int FMT, class T>
static int read_t(const ReadParams& p, cudaStream_t st) {
    const bool vec = reinterpret_cast<uintptr_t>(p.dst) % 16 == 0 && p.stride * sizeof(T) % 16 == 0;
    const dim3 grid((unsigned)((p.n + WARPS - 1) / WARPS));
    if (vec)
        read_kernel<FMT, T, true><<<grid, WARPS * 32, 0, st>>>(p);
    else
        read_kernel<FMT, T, false><<<grid, WARPS * 32, 0, st>>>(p);
    return cudaGetLastError() == cudaSuccess ? 0 : PION_B200_ECUDA;
}

}  // namespace fp4

int launch_fp4_write(const Fp4Write& w, cudaStream_t st) {
    using namespace fp4;
    if (w.n <= 0) return 0;
    if (w.slots) {
        claim_kernel<<<(unsigned)((w.n + 255) / 256), 256, 0, st>>>(w.slots, w.n, w.n_slots,
                                                                    w.claim, w.status);
        if (cudaGetLastError() != cudaSuccess) return PION_B200_ECUDA;
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
