// Microscaled 4-bit floating point: the store's layout and its element arithmetic, shared by
// the row kernels (fp4_rows.cu) and the product (flat_fp4.cu).
//
// A row is stored as e2m1 codes (sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6), two per byte, the
// lower nibble first, padded with zeros to a multiple of 128 elements; one scale byte per block
// (MX: 32 elements, e8m0; NV: 16 elements, e4m3); and one float g per row.
//
// Scale bytes lie as the tensor cores take them from TMEM: tiles of 128 rows, atoms of 4 blocks,
// 512 bytes per (tile, atom) as [row % 32][row / 32 % 4][block % 4], so that an atom is a 16-byte
// word of each of 32 lanes, four columns.
#pragma once

#include <cstdint>

#include "common.cuh"

namespace pion {
namespace fp4 {

constexpr int kMX = PION_B200_FP4_MX;
constexpr int kNV = PION_B200_FP4_NV;
// The query tile's codes and, where TMEM has no room for them, scale atoms stay in shared memory: at
// 8192 dimensions each CTA of a pair holds 64 + 64 KB of its 227 KB for 32 queries of the NV format.
constexpr int kMaxDim = 8192;

__host__ __device__ constexpr int pad_dim(int dim) { return (dim + 127) / 128 * 128; }
__host__ __device__ constexpr int block_of(int fmt) { return fmt == kMX ? 32 : 16; }
__host__ __device__ constexpr int atoms_of(int fmt, int dp) { return dp / (4 * block_of(fmt)); }

// Byte offset of the four scale bytes of (row, atom).
__host__ __device__ __forceinline__ int64_t scale_word(int64_t row, int atom, int atoms) {
    const int in = (int)(row & 127);
    return ((row >> 7) * atoms + atom) * 512 + (in & 31) * 16 + (in >> 5) * 4;
}

// A query batch is laid out in groups of `tile` queries, each group at a multiple of 128
// slots, so that a query tile's scales start at an atom.
__host__ __device__ __forceinline__ int64_t query_slot(int64_t t, int tile, int tile_pad) {
    return t / tile * tile_pad + t % tile;
}

// -------------------------------------------------- overlapped launches --
// The kernels of a call are launched with programmatic stream serialisation: a kernel may
// start while the one before it still runs, and waits for it, and for its memory, before it
// reads or writes anything.  What they read they read through L2 (never ld.global.nc): lines
// that an earlier kernel left in an SM's L1 may be older than what is waited for.
__device__ __forceinline__ void griddep_wait() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void griddep_launch() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class... P, class... A>
inline int launch_pdl(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                      const A&... args) {
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, P(args)...) == cudaSuccess ? 0 : PION_B200_ECUDA;
}

// ------------------------------------------------------------ conversions --
// Eight floats -> eight e2m1 codes (nearest, ties to even, saturating), element 0 lowest.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Eight codes -> what they stand for (exact).
__device__ __forceinline__ void e2m1x8_values(uint32_t codes, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(codes));
#pragma unroll
    for (int j = 0; j < 4; ++j)
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
            "cvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
            : "=f"(v[2 * j]), "=f"(v[2 * j + 1])
            : "r"(h[j]));
}

// Four codes (the low 16 bits) -> twice their values as signed bytes (exact integers up to
// 12): two eight-entry byte tables, |2v| and -|2v|, blended by sign.  prmt with selector bit
// 3 set replicates the chosen byte's top bit, so prmt(0x80..., codes) is 0x80 or 0xff by
// sign; shifted left it is a mask of the upper seven bits, and the lowest bit is the same in
// both tables.
__device__ __forceinline__ uint32_t e2m1x4_bytes(uint32_t codes) {
    const uint32_t sel = codes & 0x7777u;
    const uint32_t pos = __byte_perm(0x03020100u, 0x0C080604u, sel);
    const uint32_t neg = __byte_perm(0xFDFEFF00u, 0xF4F8FAFCu, sel);
    uint32_t sign;  // __byte_perm would clear the selectors' top bits
    asm("prmt.b32 %0, %1, %1, %2;" : "=r"(sign) : "r"(0x80808080u), "r"(codes & 0xFFFFu));
    const uint32_t mask = sign << 1;
    return (pos & ~mask) | (neg & mask);
}

__device__ __forceinline__ float e4m3_value(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}"
        : "=r"(h)
        : "r"(byte));
    float v;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.f32.f16 %0, lo;\n\t}"
        : "=f"(v)
        : "r"(h));
    return v;
}

// In units of 2^-9, the least of them: an integer up to 448 * 512.
__device__ __forceinline__ uint32_t e4m3_units(uint32_t byte) {
    const uint32_t e = byte >> 3, m = byte & 7u;
    return e ? (8u | m) << (e - 1u) : m;
}

// 2^(byte - 127), exact down to the subnormal 2^-127.
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
}

template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return FMT == kMX ? e8m0_value(byte) : e4m3_value(byte);
}

}  // namespace fp4
}  // namespace pion
