// MX wire format for MI355X (gfx950): element codes + one E8M0 scale byte per 32 elements.
//
// The reference ("FQ" = mor/csrc/cuda/fake_quantize.cu) only returns the dequantized bf16 tensor.  These kernels
// emit what its MX block quantization (block modes with SF_E8, FQ:801-823, E2M3 branch FQ:758-770) holds between
// "quantize" and "dequantize": per block of 32 elements, e8 = exponent field of fl32(fmax / amax) - 127 (FQ:251-252),
// code = cast(x * 2^e8), scale byte = 127 - e8 (the E8M0 encoding of the multiplier 2^-e8 that decodes the block).
//   k_mx_quantize    blocks along rows: a lane owns 8 elements, 4 lanes a block (amax by DPP), 8 or 6 bytes per lane
//   k_mx_dual        one read of a 128 x 128 tile gives both orientations: blocks along rows from registers, blocks
//                    along columns through an LDS copy of the tile, written transposed ([cols, rows] payload) so that
//                    the reduction dimension of a weight-gradient GEMM is contiguous
//   k_mx_dequantize  payload + scales -> bf16
// FP8 and FP6 codes come from the gfx950 FP8 converts (E2M3 / E3M2 share the mantissa width of E4M3 / E5M2, see
// code_pair), E2M1 codes from its scaled FP4 convert.  FP6 codes are packed little-endian, 32 codes in 24 bytes, E2M1
// codes two to a byte, 16 bytes a block.  The file also holds k_fq_dual, the fake-quantized
// tensor and the fake-quantized transpose from one read.

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>

#include "mor_common.h"
#include "mor_wirefmt.h"
#include "mor_host.h"
#include "../../include/mor_hip.h"

namespace mor {

constexpr int WWG = 256;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Exponent of the block scale, limited to the finite E8M0 range.  The integer form needs a normal amax; the
// division covers subnormal amax and the far ends of the exponent range.
// E2M1 has no code for an infinity or a NaN: a block that holds one (amax as block_amax gives it) gets E8_NONFINITE,
// whose scale byte 127 - e8 is the E8M0 NaN, and decodes to NaNs.
constexpr int E8_NONFINITE = -128;
template <int F> __device__ __forceinline__ int wire_e8(float amax) {
    if constexpr (F == FMT_E2M1) { if (f2u(amax) >= 0x7F800000u) return E8_NONFINITE; }
    if (!(amax > 0.0f)) return 0;
    const Scale sc = make_scale_e8<F>(amax);
    int e8 = sc.e8;
    if (!sc.fast) e8 = (int)((f2u(Fmt<F>::fmax / amax) >> 23) & 0xFF) - 127;
    return min(max(e8, -127), 127);
}

// The byte of two E2M1 codes of a packed word.  v_cvt_scalef32_pk_fp4_bf16 divides by its scale and rounds to nearest
// even (mor_selftest_hw_fp4 compares the two forms for every finite bf16 value and every e8 in [-126, 126]); the
// software form counts the midpoints below |x| * 2^e8, a midpoint itself going to the even code.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ bool fp4_hw_ok(int e8) { return e8 >= -126 && e8 <= 126; }
__device__ __forceinline__ uint32_t fp4_mag_code(float a) {
    return (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
}
__device__ __forceinline__ uint32_t fp4_pair_sw(uint32_t w, int e8) {
    if (e8 == E8_NONFINITE) return 0;
    const uint32_t a = fp4_mag_code(ldexpf(fabsf(bf16_lo(w)), e8)), b = fp4_mag_code(ldexpf(fabsf(bf16_hi(w)), e8));
    return a | ((w >> 12) & 8u) | ((b | ((w >> 28) & 8u)) << 4);
}
// the 8 codes of four packed words, element i in bits [4 i, 4 i + 4)
__device__ __forceinline__ uint32_t fp4_octet(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, int e8) {
    if (fp4_hw_ok(e8)) {
        const float scale = u2f((uint32_t)(127 - e8) << 23);
        uint32_t p = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf16x2, w0), scale, 0);
        p = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(p, __builtin_bit_cast(bf16x2, w1), scale, 1);
        p = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(p, __builtin_bit_cast(bf16x2, w2), scale, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(p, __builtin_bit_cast(bf16x2, w3), scale, 3);
    }
    return fp4_pair_sw(w0, e8) | (fp4_pair_sw(w1, e8) << 8) | (fp4_pair_sw(w2, e8) << 16) | (fp4_pair_sw(w3, e8) << 24);
}
// value of an E2M1 code
__device__ __forceinline__ float fp4_value(uint32_t code) {
    const uint32_t e = (code >> 1) & 3u, m = code & 1u;
    const float mag = e == 0 ? 0.5f * (float)m : u2f(((e + 126u) << 23) | (m << 22));
    return u2f(f2u(mag) | ((code & 8u) << 28));
}
// the 8 values of an octet of codes times 2^de, as bf16
__device__ __forceinline__ uint4 fp4_octet_decode_hw(uint32_t q, int de) {
    const float scale = u2f((uint32_t)(127 + de) << 23);
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, scale, 3)));
}

// codes of the two elements of a packed word, in bits 0..bits-1 and bits..2*bits-1 (FP6: fp6_mag_codes).
template <int F> __device__ __forceinline__ uint32_t code_pair(uint32_t w, int e8) {
    if constexpr (Fmt<F>::hw) {
        return hw_pack2<F>(ldexpf(bf16_lo(w), e8), ldexpf(bf16_hi(w), e8)) & 0xFFFFu;
    } else {
        // (in a block scaled by its own e8 nothing exceeds fmax; the clamp is the cast's saturation for any other use)
        const float a = fminf(ldexpf(fabsf(bf16_lo(w)), e8), Fmt<F>::fmax), b = fminf(ldexpf(fabsf(bf16_hi(w)), e8), Fmt<F>::fmax);
        uint32_t ca, cb;
        fp6_mag_codes<F>(a, b, ca, cb);
        return ca | ((w >> 10) & 0x20u) | ((cb | ((w >> 26) & 0x20u)) << 6);
    }
}

// the 8 codes of a 16-byte chunk: 64 bits (FP8) or 48 bits (FP6)
template <int F> __device__ __forceinline__ uint64_t code_chunk(uint4 v, int e8) {
    constexpr int pb = 2 * Wire<F>::bits;
    return (uint64_t)code_pair<F>(v.x, e8) | ((uint64_t)code_pair<F>(v.y, e8) << pb) |
           ((uint64_t)code_pair<F>(v.z, e8) << (2 * pb)) | ((uint64_t)code_pair<F>(v.w, e8) << (3 * pb));
}

template <int F, bool HIGH> __device__ __forceinline__ uint32_t fp8_pair_decode_hw(uint32_t codes, float scale) {
    if constexpr (F == FMT_E4M3) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)codes, scale, HIGH));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8((int)codes, scale, HIGH));
}
// the same 6 words from the software codes of 16 packed pairs
template <int F> __device__ __forceinline__ u32x6 fp6_block_sw(const uint32_t (&words)[16], int e8) {
    uint32_t p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i] = code_pair<F>(words[i], e8);
    u32x6 d;
#pragma unroll
    for (int g = 0; g < 6; ++g) {
        uint32_t acc = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int lo_bit = 12 * i - 32 * g;                      // position of pair i in this word
            if (lo_bit > -12 && lo_bit < 32) acc |= lo_bit >= 0 ? (p[i] << lo_bit) : (p[i] >> (-lo_bit));
        }
        d[g] = acc;
    }
    return d;
}

__device__ __forceinline__ float chunk_amax(uint4 v) {
    float amax = 0.0f;
    acc_amax(amax, v.x); acc_amax(amax, v.y); acc_amax(amax, v.z); acc_amax(amax, v.w);
    return amax;
}

// Largest magnitude of the block whose four chunks the lanes of a quad hold.  E2M1: of the bit patterns, so that an
// infinity or a NaN wins (the other formats carry them in their codes, and a NaN does not take part).
template <int F> __device__ __forceinline__ float block_amax(uint4 v) {
    if constexpr (F == FMT_E2M1) {
        uint32_t m = 0;
        acc_amax_pk(m, v.x); acc_amax_pk(m, v.y); acc_amax_pk(m, v.z); acc_amax_pk(m, v.w);
        return u2f(group_umax(amax_bits_of(m), 4));
    } else return group_max_t<4>(chunk_amax(v), 4);
}
// the same of 32 values in one lane
template <int F> __device__ __forceinline__ float words_amax(const uint32_t (&w)[16]) {
    if constexpr (F == FMT_E2M1) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc_amax_pk(m, w[i]);
        return u2f(amax_bits_of(m));
    } else {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc_amax(amax, w[i]);
        return amax;
    }
}

// Quantizes and stores one chunk; `c` is the chunk's index in the payload's own row-major order (4 chunks = 1 block,
// held by the 4 lanes of a quad; every lane of the quad must call this).
// FP8: 8 bytes per lane.  E2M1: 4 bytes per lane.  FP6: the quad's 16 words are broadcast to its lanes (DPP), every lane converts the whole
// block with one instruction and lanes 0..2 store 8 of the 24 bytes each; outside the range of the block convert the
// software codes are merged across the quad instead.
template <int F> __device__ __forceinline__ void emit_chunk(uint8_t* payload, int64_t c, uint4 v, int e8, bool ok) {
    if constexpr (Fmt<F>::hw) {
        const uint64_t codes = code_chunk<F>(v, e8);
        if (ok) *reinterpret_cast<uint2*>(payload + c * 8) = make_uint2((uint32_t)codes, (uint32_t)(codes >> 32));
    } else if constexpr (F == FMT_E2M1) {
        const uint32_t codes = fp4_octet(v.x, v.y, v.z, v.w, e8);
        if (ok) *reinterpret_cast<uint32_t*>(payload + c * 4) = codes;
    } else {
        const int j = (int)(c & 3);
        uint32_t lo, hi;
        if (fp6_hw_ok(e8)) {                                     // uniform over the quad (e8 is the block's)
            uint32_t w[16];
            quad_gather(v, w);
            const u32x6 d = fp6_block_hw<F>(w, e8);
            lo = j == 0 ? d[0] : j == 1 ? d[2] : d[4];
            hi = j == 0 ? d[1] : j == 1 ? d[3] : d[5];
        } else {
            const uint64_t codes = code_chunk<F>(v, e8);
            constexpr int NEXT = 0xF9;                           // quad_perm [1,2,3,3]: lane i reads lane i + 1
            const uint32_t nlo = dpp_u<NEXT>((uint32_t)codes), nhi = dpp_u<NEXT>((uint32_t)(codes >> 32));
            const uint64_t next = (uint64_t)nlo | ((uint64_t)nhi << 32);
            const uint64_t word = (codes >> (16 * j)) | (next << (48 - 16 * j));
            lo = (uint32_t)word;
            hi = (uint32_t)(word >> 32);
        }
        if (ok && j < 3) *reinterpret_cast<uint2*>(payload + (c >> 2) * 24 + j * 8) = make_uint2(lo, hi);
    }
}

// 8- and 4-bit formats, blocks whose scale exponent is within 2^+-100, which excludes zeros, infinities and NaNs: scale and
// codes in few instructions.  With amax = m 2^ea and fmax = f 2^eb, e8 = eb - ea - (m > f) (make_scale_e8), so that the
// scale byte 127 - e8 is the exponent field of amax plus the carry of (mantissa > f's), minus eb; and the byte in place of
// an exponent is the scale that the scaled converts divide by, straight from the packed bf16 words (mor_selftest_hw_cast
// and mor_selftest_hw_fp4 compare them with the other form).
template <int F> struct QuickScale {
    static constexpr uint32_t eb = F == FMT_E4M3 ? 8 : F == FMT_E5M2 ? 15 : 2, mantissa = F == FMT_E2M1 ? 0x40u : 0x60u;
    uint32_t byte;
    bool ok;
    __device__ __forceinline__ explicit QuickScale(uint32_t amax_bits) {
        byte = ((amax_bits + ((0x7Fu - mantissa) << 16)) >> 23) - eb;
        ok = byte - 27u <= 200u;
    }
    __device__ __forceinline__ float value() const { return u2f(byte << 23); }
};
__device__ __forceinline__ uint32_t octet_amax_bits(uint4 v) {
    uint32_t m = 0;
    acc_amax_pk(m, v.x); acc_amax_pk(m, v.y); acc_amax_pk(m, v.z); acc_amax_pk(m, v.w);
    return amax_bits_of(m);
}
// 4 codes of two packed words
template <int F> __device__ __forceinline__ uint32_t quick_codes8(uint32_t w0, uint32_t w1, float scale) {
    s16x2 p = {0, 0};
    if constexpr (F == FMT_E4M3) {
        p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(bf16x2, w0), scale, false);
        p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(bf16x2, w1), scale, true);
    } else {
        p = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(p, __builtin_bit_cast(bf16x2, w0), scale, false);
        p = __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(p, __builtin_bit_cast(bf16x2, w1), scale, true);
    }
    return __builtin_bit_cast(uint32_t, p);
}
__device__ __forceinline__ uint32_t quick_codes4(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, float scale) {
    uint32_t p = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, __builtin_bit_cast(bf16x2, w0), scale, 0);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(p, __builtin_bit_cast(bf16x2, w1), scale, 1);
    p = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(p, __builtin_bit_cast(bf16x2, w2), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(p, __builtin_bit_cast(bf16x2, w3), scale, 3);
}
// Quantizes and stores the chunk `c` of a block that a quad holds; returns the block's scale byte.  (Plain stores: past the
// caches they take less time from 2^27 elements on, 16384 x 14336 in E2M1 99 -> 93 us, but the decode after them more, 171
// -> 195 us for both.)
template <int F> __device__ __forceinline__ uint32_t quantize_chunk(uint8_t* payload, int64_t c, uint4 v, bool store) {
    if constexpr (Wire<F>::bits != 6) {
        const QuickScale<F> q(group_umax(octet_amax_bits(v), 4));
        if (q.ok) {                                              // uniform over the quad
            if constexpr (F == FMT_E2M1) {
                const uint32_t codes = quick_codes4(v.x, v.y, v.z, v.w, q.value());
                if (store) *reinterpret_cast<uint32_t*>(payload + c * 4) = codes;
            } else {
                const uint2 codes = make_uint2(quick_codes8<F>(v.x, v.y, q.value()), quick_codes8<F>(v.z, v.w, q.value()));
                if (store) *reinterpret_cast<uint2*>(payload + c * 8) = codes;
            }
            return q.byte;
        }
    }
    const int e8 = wire_e8<F>(block_amax<F>(v));
    emit_chunk<F>(payload, c, v, e8, store);
    return (uint32_t)(127 - e8);
}
// the scale bytes of 4 consecutive blocks (16 lanes), in the first of the lanes
__device__ __forceinline__ uint32_t gather_scales(uint32_t sb) {
    constexpr int SHL4 = 0x104, SHL8 = 0x108, SHL12 = 0x10C;     // row_shl: lane i reads lane i + 4, 8, 12 of its 16
    return sb | (dpp_u<SHL4>(sb) << 8) | (dpp_u<SHL8>(sb) << 16) | (dpp_u<SHL12>(sb) << 24);
}

// ------------------------------------------------------------------------------------------------
// blocks of 32 along rows; the tensor is a flat array of 16-byte chunks (cols % 32 == 0).  Bound by memory: 8192 x 8192 takes
// 33 to 34 us in E4M3 (6.0 to 6.2 TB/s), 27 in E2M1 (6.3 TB/s)
template <int F, int NV>
__global__ __launch_bounds__(WWG) void k_mx_quantize(const uint4* in, uint8_t* payload, uint8_t* scales, int64_t nchunks) {
    const int64_t base = (int64_t)blockIdx.x * (NV * WWG) + threadIdx.x;
    uint4 v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t c = base + k * WWG;
        v[k] = make_uint4(0, 0, 0, 0);
        if (c < nchunks) v[k] = load16_rt(in + c, streams_last_read(nchunks * 8));
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t c = base + k * WWG;
        // the scale bytes of 4 consecutive blocks (16 lanes) leave as one 32-bit store
        const uint32_t s4 = gather_scales(quantize_chunk<F>(payload, c, v[k], c < nchunks));
        if (c < nchunks && (c & 15) == 0) {
            if (c + 16 <= nchunks) *reinterpret_cast<uint32_t*>(scales + (c >> 2)) = s4;
            else
                for (int64_t b = 0; b < ((nchunks - c) >> 2); ++b) scales[(c >> 2) + b] = (uint8_t)(s4 >> (8 * b));
        }
    }
}

// ------------------------------------------------------------------------------------------------
// both orientations from one read, blocks along rows in format FR, along columns in FC.  Tile 128 rows x 128 columns;
// cols % 32 == 0.  Where rows % 32 != 0 the last block of every column is filled up with zeros.  Bound by memory, which
// takes reads of 256-byte pieces and writes of 64 (E2M1) or 128 bytes per row and column worse than a copy: 8192 x 8192 takes
// 41.7 us in E2M1 with its input in memory and 32.8 with it in the last-level cache (4.9 and 6.2 TB/s), 52.5 and 41.6 in E4M3
// (5.2 and 6.6 TB/s).  Two workgroups per CU do better than four on large tensors (see launch_dual).  Tiles of 256 rows (25 ->
// 32 us at 2080 x 14336) and the next tile's loads held in registers over the column phase (24 -> 26) were slower.
constexpr int TILE_C = 128;
constexpr int TILE_ROWS = 128;
constexpr int DUAL_THREADS = 512;

// Workgroup -> tile.  Consecutive workgroup ids go round the 8 XCDs, each with an L2 of its own, and a tile writes
// only 4 scale bytes (and, for 6-bit codes, 96 payload bytes) of each memory line it shares with its neighbours: with
// neighbours on other XCDs every L2 writes its part of the line back by itself.  So groups of 2^lw x 2^lh neighbouring
// tiles run on one XCD, where the parts meet in one L2 before they go to memory (8192 x 8192: 47.1 -> 44.6 us for
// E4M3 codes, 71 -> 65 us for the bf16 outputs; 16384 x 14336 with 6-bit codes: 265 -> 201 us).  map = lw | lh << 2,
// chosen by dual_tile_map() so that the tile grid divides into whole groups, 8 at a time; 0 = row-major order;
// 16 = one band of tiles_x / 8 tile columns per XCD (tensors beyond the last-level cache, as in k_wgblock).
struct DualMap {
    int map;
    DivU32 per_row;           // tiles, groups or a band's tiles per row of them
};
__device__ __forceinline__ void dual_tile(uint32_t b, const DualMap& t, int64_t& ty, int64_t& tx) {
    if (t.map == 16) {                // each XCD takes a band of tiles_x / 8 tile columns and walks it row by row
        const uint32_t xcd = b & 7u, j = b >> 3, y = div_u32(j, t.per_row);
        ty = y;
        tx = xcd * t.per_row.d + (j - y * t.per_row.d);
    } else if (t.map != 0) {
        const int lw = t.map & 3, lh = t.map >> 2;
        const uint32_t xcd = b & 7u, s = b >> 3, group = (s >> (lw + lh)) * 8 + xcd, within = s & ((1u << (lw + lh)) - 1u);
        const uint32_t gy = div_u32(group, t.per_row), gx = group - gy * t.per_row.d;
        ty = (gy << lh) + (within >> lw);
        tx = (gx << lw) + (within & ((1u << lw) - 1u));
    } else {
        const uint32_t y = div_u32(b, t.per_row);
        ty = y;
        tx = b - y * t.per_row.d;
    }
}

// (tiles_x * tiles_y < 2^31)
static DualMap dual_tile_map(int64_t tiles_x, int64_t tiles_y) {
    // tensors beyond the 256 MB last-level cache: bands (16384 x 14336: E4M3 196 -> 190 us, bf16 outputs 302 -> 293 us)
    if (tiles_x % 8 == 0 && tiles_x * tiles_y > ((int64_t)128 << 20) / (TILE_ROWS * TILE_C)) return {16, make_div((uint32_t)(tiles_x / 8))};
    static const int shapes[][2] = {{3, 3}, {3, 2}, {2, 3}, {2, 2}, {3, 1}, {3, 0}, {2, 0}};      // log2 width, log2 height
    for (const auto& sh : shapes) {
        const int64_t gw = (int64_t)1 << sh[0], gh = (int64_t)1 << sh[1];
        if (tiles_x % gw == 0 && tiles_y % gh == 0 && ((tiles_x / gw) * (tiles_y / gh)) % 8 == 0) return {sh[0] | (sh[1] << 2), make_div((uint32_t)(tiles_x / gw))};
    }
    // (bands too where no group divides the grid: 2080 x 14336 in E2M1 22.4 -> 19.9 us)
    if (tiles_x % 8 == 0) return {16, make_div((uint32_t)(tiles_x / 8))};
    return {0, make_div((uint32_t)tiles_x)};
}

template <int FR, int FC>
__global__ __launch_bounds__(DUAL_THREADS) void k_mx_dual(const uint4* in, uint8_t* row_payload, uint8_t* row_scales,
                                                 uint8_t* col_payload, uint8_t* col_scales, int64_t rows, int64_t cols, DualMap map) {
    constexpr int TR = TILE_ROWS, DT = DUAL_THREADS;
    constexpr int NV = TR * (TILE_C / 8) / DT;   // 16-byte chunks per thread
    constexpr int RB = TR / 32;                   // row blocks per tile column
    constexpr int BPT = TILE_C * RB / DT;        // column blocks per thread
    constexpr int blk_bytes = 32 * Wire<FC>::bits / 8;
    constexpr int SEG = blk_bytes % 16 == 0 ? 16 : 8;      // bytes per lane of the column stores (both divide blk_bytes)
    constexpr int CODE_PITCH = (RB * blk_bytes + 16 + 15) / 16 * 16;   // bytes per column of the code tile (padded, 16-byte aligned)
    constexpr int SEGS = RB * blk_bytes / SEG;    // per column
    // one buffer, two uses: the bf16 tile, then the codes of the column blocks (smaller)
    __shared__ __attribute__((aligned(16))) uint16_t tile[TR * TILE_C];
    static_assert(RB == 4, "the column blocks' scale bytes leave as one word");
    __shared__ __attribute__((aligned(4))) uint8_t s_cscale[TILE_C * RB];
    uint8_t* codes = reinterpret_cast<uint8_t*>(tile);
    static_assert(TILE_C * CODE_PITCH <= TR * TILE_C * 2, "the code tile must fit the bf16 tile");
    const int tid = threadIdx.x;
    int64_t ty, tx;
    dual_tile(blockIdx.x, map, ty, tx);
    const int64_t R0 = ty * TR, C0 = tx * TILE_C;
    const int rows_valid = (int)min((int64_t)TR, rows - R0), cols_valid = (int)min((int64_t)TILE_C, cols - C0);
    const int64_t row_chunks = cols >> 3;

    // chunk k of a thread: row (tid >> 4) + k DT / 16 of the tile, columns 8 (tid & 15) ..
    constexpr int STEP = DT / 16;
    const int r0 = tid >> 4, cc = tid & 15;
    const int64_t first = (R0 + r0) * row_chunks + (C0 >> 3) + cc, step = STEP * row_chunks;       // as chunks of the tensor
    const bool full = rows_valid == TR && cols_valid == TILE_C;            // the same in every lane
    uint4 v[NV];
    if (full) {
        // Inputs of 192 to 256 MiB, which fill the last-level cache by themselves, are read past the caches: written or read just
        // before, 8192 x 14336 E4M3 takes 79 instead of 91 us (99.5 and 96 from memory), 16384 x 8192 90 and 103 (108 and 104),
        // 12288 x 8192 67 and 72 (81 and 78).  Smaller ones stay there for the most part: 8192 x 8192 E4M3 47.1 us past the
        // caches, 41.6 through them (53.6 and 52.5), E2M3 48.5 and 42.0 (51.0 and 51.7), 10240 x 8192 56.4 and 51.0 (63.5 and
        // 62.7).  Of larger ones little does: 16384 x 14336 E4M3 205 and 193 (205 and 190), E2M3 178 and 186 (189 and 183).
        const int64_t n = rows * cols;
        load16_group(v, n >= ((int64_t)3 << 25) && n <= ((int64_t)1 << 27), [&](int k) { return in + first + k * step; });
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            v[k] = make_uint4(0, 0, 0, 0);
            if (r0 + k * STEP < rows_valid && cc * 8 < cols_valid) v[k] = in[first + k * step];
        }
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) *reinterpret_cast<uint4*>(&tile[(r0 + k * STEP) * TILE_C + (((cc >> 2) ^ (r0 & 3)) * 32) + (cc & 3) * 8]) = v[k];
    // blocks along rows, from registers, before the columns are read back: their registers are free by then (71 -> 43).
    // The 8-bit transposed payload is streamed out while the input fits the 256 MB last-level cache (measured 49.5 -> 44.9 us
    // at 8192^2); beyond that everything streams anyway and plain stores are faster.  6-bit codes keep plain stores: a
    // tile's part of a column is 96 bytes, three quarters of a memory line, and streamed parts reach memory before the
    // neighbouring tile's part joins them (8192^2: 49.4 us streamed, 47.3 plain; 16384 x 14336: 265 against 201 us).  So do
    // E2M1 codes, 64 bytes: 2080 x 14336 20.4 -> 19.2 us streamed, but the two decodes after it 23 -> 28.
    const bool nt = Wire<FC>::bits == 8 && streams_out(rows * cols) && rows * cols <= ((int64_t)128 << 20);
    if (full && (cols & 127) == 0) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t at = first + k * step;
            const uint32_t s4 = gather_scales(quantize_chunk<FR>(row_payload, at, v[k], true));
            if (cc == 0) *reinterpret_cast<uint32_t*>(row_scales + (at >> 2)) = s4;
        }
    } else {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int64_t at = first + k * step;
            const bool ok = r0 + k * STEP < rows_valid && cc * 8 < cols_valid;
            const uint32_t sb = quantize_chunk<FR>(row_payload, at, v[k], ok);
            if (ok && (cc & 3) == 0) row_scales[at >> 2] = (uint8_t)sb;
        }
    }
    __syncthreads();
    // blocks along columns: a thread owns one column and BPT row blocks of 32, read from the LDS copy by the transposing
    // read (16 lanes give 4 rows of 16 columns, each lane gets one column's 4 rows).  The 64-byte quarters of a row lie in
    // an order that changes from row to row, so that 4 rows of 32 columns cover the banks once.
    const int c = tid & (TILE_C - 1);
    const int from = ((tid & 15) >> 2) * TILE_C + (((c >> 5) ^ ((tid & 15) >> 2)) * 32) + (tid & 16) + (tid & 3) * 4;
    uint32_t w[BPT][16];
#pragma unroll
    for (int h = 0; h < BPT; ++h) {
        const int rb = (tid >> 7) * BPT + h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const s16x4 q = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)&tile[(rb * 32 + 4 * i) * TILE_C + from]);
            const uint2 p = __builtin_bit_cast(uint2, q);
            w[h][2 * i] = p.x;
            w[h][2 * i + 1] = p.y;
        }
    }
    __syncthreads();                              // every thread has its column blocks in registers: reuse the buffer

#pragma unroll
    for (int h = 0; h < BPT; ++h) {
        const int rb = (tid >> 7) * BPT + h;
        uint8_t* dst = codes + c * CODE_PITCH + rb * blk_bytes;
        if constexpr (Wire<FC>::bits != 6) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) acc_amax_pk(m, w[h][i]);
            const QuickScale<FC> quick(amax_bits_of(m));
            if (quick.ok) {
                const float scale = quick.value();
                s_cscale[c * RB + rb] = (uint8_t)quick.byte;
                if constexpr (FC == FMT_E2M1) {
                    uint32_t q[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[i] = quick_codes4(w[h][4 * i], w[h][4 * i + 1], w[h][4 * i + 2], w[h][4 * i + 3], scale);
                    *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
                } else {
                    uint32_t q[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[i] = quick_codes8<FC>(w[h][2 * i], w[h][2 * i + 1], scale);
                    *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
                    *reinterpret_cast<uint4*>(dst + 16) = make_uint4(q[4], q[5], q[6], q[7]);
                }
                continue;
            }
        }
        const int e8 = wire_e8<FC>(words_amax<FC>(w[h]));
        s_cscale[c * RB + rb] = (uint8_t)(127 - e8);
        if constexpr (Fmt<FC>::hw) {
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i] = code_pair<FC>(w[h][2 * i], e8) | (code_pair<FC>(w[h][2 * i + 1], e8) << 16);
            *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
            *reinterpret_cast<uint4*>(dst + 16) = make_uint4(q[4], q[5], q[6], q[7]);
        } else if constexpr (FC == FMT_E2M1) {
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = fp4_octet(w[h][4 * i], w[h][4 * i + 1], w[h][4 * i + 2], w[h][4 * i + 3], e8);
            *reinterpret_cast<uint4*>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
        } else {
            const u32x6 d = fp6_hw_ok(e8) ? fp6_block_hw<FC>(w[h], e8) : fp6_block_sw<FC>(w[h], e8);
            *reinterpret_cast<uint2*>(dst) = make_uint2(d[0], d[1]);
            *reinterpret_cast<uint2*>(dst + 8) = make_uint2(d[2], d[3]);
            *reinterpret_cast<uint2*>(dst + 16) = make_uint2(d[4], d[5]);
        }
    }
    __syncthreads();

    // the transposed payload: a column of the tile is RB * blk_bytes contiguous bytes, SEGS lanes store one column
    const int64_t col_row_bytes = (rows + 31) / 32 * blk_bytes;                 // bytes per column in the transposed payload
    const int valid_bytes = (rows_valid + 31) / 32 * blk_bytes;
    if (SEG == 16 || ((col_row_bytes & 15) == 0 && rows_valid == TR)) {      // 16 bytes per lane wherever they are aligned
        constexpr int S16 = RB * blk_bytes / 16;
#pragma unroll
        for (int i = 0; i < (TILE_C * S16 + DT - 1) / DT; ++i) {
            const int idx = i * DT + tid, col = idx / S16, seg = idx % S16;
            if (col < cols_valid && seg * 16 < valid_bytes && idx < TILE_C * S16)
                store16_rt(reinterpret_cast<uint4*>(col_payload + (C0 + col) * col_row_bytes + (R0 / 32) * blk_bytes + seg * 16),
                           *reinterpret_cast<const uint4*>(codes + col * CODE_PITCH + seg * 16), nt);
        }
    } else {
#pragma unroll
        for (int i = 0; i < TILE_C * SEGS / DT; ++i) {
            const int idx = i * DT + tid, col = idx / SEGS, seg = idx % SEGS;
            if (col < cols_valid && seg * SEG < valid_bytes)
                *reinterpret_cast<uint2*>(col_payload + (C0 + col) * col_row_bytes + (R0 / 32) * blk_bytes + seg * SEG) =
                    *reinterpret_cast<const uint2*>(codes + col * CODE_PITCH + seg * SEG);
        }
    }
    // scale bytes of the column blocks: RB per column and tile
    if (tid < TILE_C && c < cols_valid) {
        const uint32_t sall = *reinterpret_cast<const uint32_t*>(&s_cscale[c * RB]);
        uint8_t* dst = col_scales + (C0 + c) * ((rows + 31) / 32) + R0 / 32;
        if ((rows & 127) == 0) *reinterpret_cast<uint32_t*>(dst) = sall;
        else
            for (int b = 0; b < (rows_valid + 31) / 32; ++b) dst[b] = (uint8_t)(sall >> (8 * b));
    }
}

// ------------------------------------------------------------------------------------------------
// Fake quantization of both orientations from one read: what mor_fake_quantize returns for the tensor with 1 x 32
// blocks and for its transpose with 1 x 32 blocks (FQ:801-823 per block), the second written transposed.  Same tile
// scheme as k_mx_dual with bf16 outputs: 2 bytes read and 4 written per element instead of 8 + a transpose.
// Blocks outside the fast exponent range take the exact path in a non-unrolled loop.
template <int F, bool E8> __device__ __forceinline__ Scale block_scale(float amax) {
    if constexpr (E8) return make_scale_e8<F>(amax);
    else return make_scale(Fmt<F>::fmax / amax);
}

template <int F, bool E8>
__global__ __launch_bounds__(WWG) void k_fq_dual(const uint4* in, uint4* out_rows, int32_t* meta_rows, uint16_t* out_cols,
                                                 int32_t* meta_cols, int64_t rows, int64_t cols, int meta_val, DualMap map) {
    constexpr int TR = 128;
    constexpr int PITCH = TILE_C + 8;             // bf16 elements per LDS row (both uses of the buffer)
    constexpr int NV = TR * (TILE_C / 8) / WWG;   // 8
    constexpr int BPT = 2;                        // column blocks per thread
    __shared__ __attribute__((aligned(16))) uint16_t tile[TR * PITCH];
    const int tid = threadIdx.x;
    int64_t ty, tx;
    dual_tile(blockIdx.x, map, ty, tx);
    const int64_t R0 = ty * TR, C0 = tx * TILE_C;
    const int rows_valid = (int)min((int64_t)TR, rows - R0), cols_valid = (int)min((int64_t)TILE_C, cols - C0);
    const int64_t row_chunks = cols >> 3;

    uint4 v[NV];
    bool ok[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int ch = k * WWG + tid, r = ch >> 4, cc = ch & 15;
        ok[k] = (r < rows_valid) && (cc * 8 < cols_valid);
        v[k] = make_uint4(0, 0, 0, 0);
        if (ok[k]) v[k] = in[(R0 + r) * row_chunks + (C0 >> 3) + cc];
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int ch = k * WWG + tid, r = ch >> 4, cc = ch & 15;
        *reinterpret_cast<uint4*>(&tile[r * PITCH + cc * 8]) = v[k];
    }
    __syncthreads();
    const int c = tid & (TILE_C - 1);
    uint32_t w[BPT][16];
#pragma unroll
    for (int h = 0; h < BPT; ++h) {
        const int rb = (tid >> 7) * BPT + h;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            w[h][i] = (uint32_t)tile[(rb * 32 + 2 * i) * PITCH + c] | ((uint32_t)tile[(rb * 32 + 2 * i + 1) * PITCH + c] << 16);
    }
    // blocks along rows, from registers
    const bool nt = streams_out(rows * cols);
    uint32_t slow = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int ch = k * WWG + tid, r = ch >> 4, cc = ch & 15;
        const float amax = group_max_t<4>(chunk_amax(v[k]), 4);
        const Scale sc = block_scale<F, E8>(amax);
        const bool quant = (amax > 0.0f) && sc.fast;
        const uint4 q = fq_vec_fast<F, E8>(v[k], sc);
        uint4 o;
        o.x = quant ? q.x : v[k].x; o.y = quant ? q.y : v[k].y; o.z = quant ? q.z : v[k].z; o.w = quant ? q.w : v[k].w;
        if ((amax > 0.0f) && !sc.fast) slow |= 1u << k;
        const int64_t cidx = (R0 + r) * row_chunks + (C0 >> 3) + cc;
        if (ok[k]) {
            store16_rt(out_rows + cidx, o, nt);
            if (meta_rows && (cc & 3) == 0) meta_rows[cidx >> 2] = meta_val;
        }
    }
    if (slow) {
#pragma unroll 1
        for (int k = 0; k < NV; ++k) {
            if (!((slow >> k) & 1u)) continue;                       // uniform over the 4 lanes of a block
            const int ch = k * WWG + tid, r = ch >> 4, cc = ch & 15;
            const uint4 x = *reinterpret_cast<const uint4*>(&tile[r * PITCH + cc * 8]);
            const float amax = group_max_t<4>(chunk_amax(x), 4);
            const Scale sc = make_scale(Fmt<F>::fmax / amax);
            uint4 o;
            o.x = fq_pair_exact<F, E8, false>(x.x, sc); o.y = fq_pair_exact<F, E8, false>(x.y, sc);
            o.z = fq_pair_exact<F, E8, false>(x.z, sc); o.w = fq_pair_exact<F, E8, false>(x.w, sc);
            if (ok[k]) out_rows[(R0 + r) * row_chunks + (C0 >> 3) + cc] = o;
        }
    }
    __syncthreads();                              // every thread has its column blocks in registers: reuse the buffer

    // blocks along columns; results go to LDS transposed (PITCH elements per column, 128 of them used)
    int32_t col_meta_ok = 0;
#pragma unroll
    for (int h = 0; h < BPT; ++h) {
        const int rb = (tid >> 7) * BPT + h;
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc_amax(amax, w[h][i]);
        const Scale sc = block_scale<F, E8>(amax);
        uint32_t q[16];
        if ((amax > 0.0f) && !sc.fast) {
            const Scale se = make_scale(Fmt<F>::fmax / amax);
#pragma unroll 1
            for (int i = 0; i < 16; ++i) q[i] = fq_pair_exact<F, E8, false>(w[h][i], se);
        } else {
            const bool quant = amax > 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t f = fq_pair_fast<F, E8>(w[h][i], sc);
                q[i] = quant ? f : w[h][i];
            }
        }
        uint4* dst = reinterpret_cast<uint4*>(&tile[c * PITCH + rb * 32]);
        dst[0] = make_uint4(q[0], q[1], q[2], q[3]);
        dst[1] = make_uint4(q[4], q[5], q[6], q[7]);
        dst[2] = make_uint4(q[8], q[9], q[10], q[11]);
        dst[3] = make_uint4(q[12], q[13], q[14], q[15]);
        col_meta_ok |= (c < cols_valid && rb * 32 < rows_valid) ? (1 << h) : 0;
    }
    __syncthreads();
    // transposed output: a column of the tile is 256 contiguous bytes, 16 lanes store one column
#pragma unroll
    for (int i = 0; i < TILE_C * 16 / WWG; ++i) {
        const int idx = i * WWG + tid, col = idx >> 4, seg = idx & 15;
        if (col < cols_valid && seg * 8 < rows_valid)
            store16_rt(reinterpret_cast<uint4*>(out_cols + (C0 + col) * rows + R0 + seg * 8), *reinterpret_cast<const uint4*>(&tile[col * PITCH + seg * 8]), nt);
    }
    if (meta_cols) {
#pragma unroll
        for (int h = 0; h < BPT; ++h)
            if ((col_meta_ok >> h) & 1) meta_cols[(C0 + c) * (rows / 32) + R0 / 32 + (tid >> 7) * BPT + h] = meta_val;
    }
}

// ------------------------------------------------------------------------------------------------
template <int F>
__global__ __launch_bounds__(WWG) void k_mx_dequantize(const uint8_t* payload, const uint8_t* scales, uint4* out, int64_t nchunks) {
    for (int64_t c = (int64_t)blockIdx.x * WWG + threadIdx.x; c < nchunks; c += (int64_t)gridDim.x * WWG) {
        const int de = (int)scales[c >> 2] - 127;
        float x[8];
        if constexpr (Fmt<F>::hw) {
            const uint2 q = *reinterpret_cast<const uint2*>(payload + c * 8);
            if (fp6_decode_hw_ok(de)) {          // v_cvt_scalef32_pk_bf16_{fp8,bf8}: two codes -> two bf16 of decode * 2^de
                const float scale = u2f((uint32_t)(127 + de) << 23);
                uint4 r;
                r.x = fp8_pair_decode_hw<F, false>(q.x, scale); r.y = fp8_pair_decode_hw<F, true>(q.x, scale);
                r.z = fp8_pair_decode_hw<F, false>(q.y, scale); r.w = fp8_pair_decode_hw<F, true>(q.y, scale);
                store16_rt(out + c, r, streams_out(nchunks * 8));
                continue;
            }
            x[0] = hw_unpack<F, 0>(q.x); x[1] = hw_unpack<F, 1>(q.x); x[2] = hw_unpack<F, 2>(q.x); x[3] = hw_unpack<F, 3>(q.x);
            x[4] = hw_unpack<F, 0>(q.y); x[5] = hw_unpack<F, 1>(q.y); x[6] = hw_unpack<F, 2>(q.y); x[7] = hw_unpack<F, 3>(q.y);
        } else if constexpr (F == FMT_E2M1) {
            const uint32_t q = *reinterpret_cast<const uint32_t*>(payload + c * 4);
            if (fp6_decode_hw_ok(de)) {          // v_cvt_scalef32_pk_bf16_fp4
                store16_rt(out + c, fp4_octet_decode_hw(q, de), streams_out(nchunks * 8));
                continue;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fp4_value(q >> (4 * i));
        } else {
            if (fp6_decode_hw_ok(de)) {
                // every lane of the quad reads its block's 24 bytes (same addresses: one fetch) and decodes all 32 codes
                // with one block convert, then keeps its own 8 values
                const uint2* blk = reinterpret_cast<const uint2*>(payload + (c >> 2) * 24);
                const uint2 b0 = blk[0], b1 = blk[1], b2 = blk[2];
                const u32x16 t = fp6_block_decode_hw<F>(u32x6{b0.x, b0.y, b1.x, b1.y, b2.x, b2.y}, de);
                const int j = (int)(c & 3);
                uint4 r;
                r.x = j == 0 ? t[0] : j == 1 ? t[4] : j == 2 ? t[8] : t[12];
                r.y = j == 0 ? t[1] : j == 1 ? t[5] : j == 2 ? t[9] : t[13];
                r.z = j == 0 ? t[2] : j == 1 ? t[6] : j == 2 ? t[10] : t[14];
                r.w = j == 0 ? t[3] : j == 1 ? t[7] : j == 2 ? t[11] : t[15];
                store16_rt(out + c, r, streams_out(nchunks * 8));
                continue;
            }
            const uint16_t* p = reinterpret_cast<const uint16_t*>(payload + (c >> 2) * 24 + (c & 3) * 6);
            const uint64_t bits = (uint64_t)p[0] | ((uint64_t)p[1] << 16) | ((uint64_t)p[2] << 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t code = (uint32_t)(bits >> (6 * i)) & 0x3Fu;
                x[i] = u2f(f2u(fp6_value<F>(code & 0x1Fu)) | ((code & 0x20u) << 26));
            }
        }
        if (de == 128) {                         // scale byte 255, the E8M0 NaN (the product takes it so too)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = u2f(0x7FC00000u);
        }
        uint4 r;
        r.x = store_pair<true>(ldexpf(x[0], de), ldexpf(x[1], de));
        r.y = store_pair<true>(ldexpf(x[2], de), ldexpf(x[3], de));
        r.z = store_pair<true>(ldexpf(x[4], de), ldexpf(x[5], de));
        r.w = store_pair<true>(ldexpf(x[6], de), ldexpf(x[7], de));
        store16_rt(out + c, r, streams_out(nchunks * 8));
    }
}

// Every bf16 value x every scale exponent the block convert is used with: hardware codes against software codes.
// One thread per (32 consecutive bf16 patterns, e8); counts the differing codes.
template <int F>
__global__ __launch_bounds__(WWG) void k_selftest_hw_fp6(unsigned long long* mismatches) {
    const uint32_t idx = blockIdx.x * WWG + threadIdx.x;
    if (idx >= 2048u * 253u) return;
    const uint32_t group = idx & 2047u;
    const int e8 = (int)(idx >> 11) - 126;
    uint32_t words[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        uint32_t lo = group * 32u + 2u * i, hi = lo + 1u;
        if ((lo & 0x7F80u) == 0x7F80u) lo = 0;                   // Inf / NaN patterns are outside the contract
        if ((hi & 0x7F80u) == 0x7F80u) hi = 0;
        words[i] = lo | (hi << 16);
    }
    const u32x6 a = fp6_block_hw<F>(words, e8), b = fp6_block_sw<F>(words, e8);
    unsigned bad = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const int bit = 6 * j, g = bit >> 5, sh = bit & 31;
        uint32_t x = (a[g] ^ b[g]) >> sh;
        if (sh > 26 && g < 5) x |= (a[g + 1] ^ b[g + 1]) << (32 - sh);
        bad += (x & 0x3Fu) != 0;
    }
    if (bad) atomicAdd(mismatches + F, (unsigned long long)bad);
}

// The inverse convert: the 64 codes (two groups of 32) with every scale exponent it is used with.
template <int F>
__global__ __launch_bounds__(WWG) void k_selftest_hw_fp6_decode(unsigned long long* mismatches) {
    const int idx = blockIdx.x * WWG + threadIdx.x;
    if (idx >= 2 * 201) return;
    const int half = idx & 1, de = (idx >> 1) - 100;
    uint32_t d[6] = {0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const uint64_t code = (uint64_t)(half * 32 + j) << ((6 * j) & 31);
        d[(6 * j) >> 5] |= (uint32_t)code;
        if (((6 * j) >> 5) < 5) d[((6 * j) >> 5) + 1] |= (uint32_t)(code >> 32);
    }
    const u32x16 t = fp6_block_decode_hw<F>(u32x6{d[0], d[1], d[2], d[3], d[4], d[5]}, de);
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint32_t c0 = half * 32 + 2 * i, c1 = c0 + 1;
        const float v0 = u2f(f2u(fp6_value<F>(c0 & 0x1Fu)) | ((c0 & 0x20u) << 26)), v1 = u2f(f2u(fp6_value<F>(c1 & 0x1Fu)) | ((c1 & 0x20u) << 26));
        const uint32_t want = store_pair<true>(ldexpf(v0, de), ldexpf(v1, de));
        bad += ((t[i] ^ want) & 0xFFFFu) != 0;
        bad += ((t[i] ^ want) >> 16) != 0;
    }
    if (bad) atomicAdd(mismatches + F, (unsigned long long)bad);
}

// v_cvt_scalef32_pk_bf16_{fp8,bf8} (dequantize): the 254 finite-or-not codes as they come, every scale exponent used.
template <int F>
__global__ __launch_bounds__(WWG) void k_selftest_hw_fp8_decode(unsigned long long* mismatches) {
    const int idx = blockIdx.x * WWG + threadIdx.x;
    if (idx >= 128 * 201) return;
    const uint32_t c0 = 2u * (idx & 127), c1 = c0 + 1u;
    const int de = (idx >> 7) - 100;
    const float v0 = hw_unpack<F, 0>(c0 | (c1 << 8)), v1 = hw_unpack<F, 1>(c0 | (c1 << 8));
    if (v0 != v0 || v1 != v1 || fabsf(v0) > Fmt<F>::fmax || fabsf(v1) > Fmt<F>::fmax) return;     // NaN / Inf codes are never produced
    const uint32_t want = store_pair<true>(ldexpf(v0, de), ldexpf(v1, de));
    const uint32_t got = fp8_pair_decode_hw<F, false>(c0 | (c1 << 8), u2f((uint32_t)(127 + de) << 23));
    const uint32_t got_hi = fp8_pair_decode_hw<F, true>((c0 | (c1 << 8)) << 16, u2f((uint32_t)(127 + de) << 23));
    const unsigned bad = (got != want) + (got_hi != want);
    if (bad) atomicAdd(mismatches + F, (unsigned long long)bad);
}

// E2M1 converts: mismatches[0], every bf16 pair of patterns x every scale exponent the hardware convert is used with;
// mismatches[1], the 16 codes (two octets) x every scale exponent of the decode.
__global__ __launch_bounds__(WWG) void k_selftest_hw_fp4(unsigned long long* mismatches) {
    const uint32_t idx = blockIdx.x * WWG + threadIdx.x;
    if (idx >= 8192u * 253u) return;
    const int e8 = (int)(idx >> 13) - 126;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (idx & 8191u) * 8u + 2u * i;
        w[i] = (lo & 0x7F80u) == 0x7F80u ? 0u : lo | ((lo + 1u) << 16);          // Inf / NaN blocks never reach the convert
    }
    const uint32_t want = fp4_pair_sw(w[0], e8) | (fp4_pair_sw(w[1], e8) << 8) | (fp4_pair_sw(w[2], e8) << 16) | (fp4_pair_sw(w[3], e8) << 24);
    if (fp4_octet(w[0], w[1], w[2], w[3], e8) != want) atomicAdd(mismatches, 1ull);
}
__global__ __launch_bounds__(WWG) void k_selftest_hw_fp4_decode(unsigned long long* mismatches) {
    const int idx = blockIdx.x * WWG + threadIdx.x;
    if (idx >= 2 * 201) return;
    const int de = (idx >> 1) - 100;
    const uint32_t q = (idx & 1) ? 0xFEDCBA98u : 0x76543210u;
    const uint4 got = fp4_octet_decode_hw(q, de);
    const uint32_t r[4] = {got.x, got.y, got.z, got.w};
    unsigned bad = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad += r[i] != store_pair<true>(ldexpf(fp4_value(q >> (8 * i)), de), ldexpf(fp4_value(q >> (8 * i + 4)), de));
    if (bad) atomicAdd(mismatches + 1, (unsigned long long)bad);
}

}  // namespace mor

using namespace mor;

static int validate_wire(const void* a, const void* b, const void* c, int64_t rows, int64_t cols, int fmt, int64_t row_multiple) {
    if (!a || !b || !c) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
    if (rows <= 0 || cols <= 0) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "rows and cols must be positive (got %lld x %lld)", (long long)rows, (long long)cols);
    if (cols % 32 || rows % row_multiple)
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "MX blocks need cols %% 32 == 0 and rows %% %lld == 0 (got %lld x %lld)", (long long)row_multiple, (long long)rows, (long long)cols);
    if (fmt < MOR_FMT_E4M3 || fmt > MOR_FMT_E2M1) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "unknown element format %d", fmt);
    if (rows > MOR_MAX_ELEMENTS / cols) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensor too large (more than 2^35 elements)");
    if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15u) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensor and payload must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(c) & 3u) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "scales must be 4-byte aligned");
    return MOR_OK;
}

extern "C" size_t mor_mx_payload_bytes(int64_t rows, int64_t cols, int fmt) {
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)rows * (size_t)cols * ((fmt == MOR_FMT_E4M3 || fmt == MOR_FMT_E5M2) ? 8 : fmt == MOR_FMT_E2M1 ? 4 : 6) / 8;
}

extern "C" int mor_mx_quantize(const void* input, void* payload, void* scales, int64_t rows, int64_t cols, int fmt, void* stream) {
    if (int rc = validate_wire(input, payload, scales, rows, cols, fmt, 1)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t nchunks = rows * cols / 8;
    constexpr int NV = 2;
    const unsigned grid = (unsigned)((nchunks + NV * WWG - 1) / (NV * WWG));
    const uint4* in = static_cast<const uint4*>(input);
    uint8_t* p = static_cast<uint8_t*>(payload);
    uint8_t* s = static_cast<uint8_t*>(scales);
    switch (fmt) {
        case MOR_FMT_E4M3: k_mx_quantize<FMT_E4M3, NV><<<grid, WWG, 0, st>>>(in, p, s, nchunks); break;
        case MOR_FMT_E5M2: k_mx_quantize<FMT_E5M2, NV><<<grid, WWG, 0, st>>>(in, p, s, nchunks); break;
        case MOR_FMT_E2M1: k_mx_quantize<FMT_E2M1, NV><<<grid, WWG, 0, st>>>(in, p, s, nchunks); break;
        case MOR_FMT_E3M2: k_mx_quantize<FMT_E3M2, NV><<<grid, WWG, 0, st>>>(in, p, s, nchunks); break;
        default: k_mx_quantize<FMT_E2M3, NV><<<grid, WWG, 0, st>>>(in, p, s, nchunks); break;
    }
    return mor_check_launch("k_mx_quantize");
}

template <int FR, int FC>
static int launch_dual(const void* input, void* row_payload, void* row_scales, void* col_payload, void* col_scales, int64_t rows,
                       int64_t cols, hipStream_t st) {
    const int64_t tiles_y = (rows + TILE_ROWS - 1) / TILE_ROWS, tiles_x = (cols + TILE_C - 1) / TILE_C;
    // (a grid of 2^32 threads would be cut without an error: one tile column of 2^30 rows)
    if (tiles_y * tiles_x >= (1ll << 32) / DUAL_THREADS) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "too many tiles");
    // From 2^25 elements on, LDS that is not used keeps a third workgroup off a CU.  8192 x 8192, input in memory: E2M1 46.1 ->
    // 41.7 us, E4M3 56.5 -> 52.3, E2M3 56.4 -> 51.7; in the last-level cache 33.6 -> 32.8, 42.0 -> 41.6, 41.5 -> 41.8; 16384 x
    // 14336 E2M1 167 -> 145, E4M3 197 -> 190; 8192 x 4096 E4M3 30.3 -> 29.6 and 21.7 -> 22.8.  Below, 4096 x 4096, 10.6 -> 11.9.
    const unsigned spare = rows * cols >= ((int64_t)1 << 25) ? 40000u : 0u;
    k_mx_dual<FR, FC><<<(unsigned)(tiles_y * tiles_x), DUAL_THREADS, spare, st>>>(
        static_cast<const uint4*>(input), static_cast<uint8_t*>(row_payload), static_cast<uint8_t*>(row_scales),
        static_cast<uint8_t*>(col_payload), static_cast<uint8_t*>(col_scales), rows, cols, dual_tile_map(tiles_x, tiles_y));
    return mor_check_launch("k_mx_dual");
}

extern "C" int mor_mx_quantize_dual(const void* input, void* row_payload, void* row_scales, void* col_payload, void* col_scales,
                                    int64_t rows, int64_t cols, int fmt, void* stream) {
    if (int rc = validate_wire(input, row_payload, row_scales, rows, cols, fmt, 32)) return rc;
    if (int rc = validate_wire(input, col_payload, col_scales, rows, cols, fmt, 32)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (fmt) {
        case MOR_FMT_E4M3: return launch_dual<FMT_E4M3, FMT_E4M3>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
        case MOR_FMT_E5M2: return launch_dual<FMT_E5M2, FMT_E5M2>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
        case MOR_FMT_E3M2: return launch_dual<FMT_E3M2, FMT_E3M2>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
        case MOR_FMT_E2M3: return launch_dual<FMT_E2M3, FMT_E2M3>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
        default: return launch_dual<FMT_E2M1, FMT_E2M1>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
    }
}

extern "C" int mor_mx_quantize_dual_ragged(const void* input, void* row_payload, void* row_scales, void* col_payload, void* col_scales,
                                           int64_t rows, int64_t cols, int row_fmt, int col_fmt, void* stream) {
    if (int rc = validate_wire(input, row_payload, row_scales, rows, cols, row_fmt, 1)) return rc;
    if (int rc = validate_wire(input, col_payload, col_scales, rows, cols, col_fmt, 1)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (row_fmt == MOR_FMT_E4M3 && col_fmt == MOR_FMT_E4M3) return launch_dual<FMT_E4M3, FMT_E4M3>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
    if (row_fmt == MOR_FMT_E5M2 && col_fmt == MOR_FMT_E5M2) return launch_dual<FMT_E5M2, FMT_E5M2>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
    if (row_fmt == MOR_FMT_E2M1 && col_fmt == MOR_FMT_E2M1) return launch_dual<FMT_E2M1, FMT_E2M1>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
    if (row_fmt == MOR_FMT_E2M1 && col_fmt == MOR_FMT_E4M3) return launch_dual<FMT_E2M1, FMT_E4M3>(input, row_payload, row_scales, col_payload, col_scales, rows, cols, st);
    return mor_fail(MOR_ERR_INVALID_ARGUMENT, "formats %d along rows and %d along columns: one of E4M3, E5M2, E2M1 for both, or E2M1 and E4M3", row_fmt, col_fmt);
}

extern "C" int mor_mx_dequantize(const void* payload, const void* scales, void* output, int64_t rows, int64_t cols, int fmt, void* stream) {
    if (int rc = validate_wire(output, payload, scales, rows, cols, fmt, 1)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t nchunks = rows * cols / 8;
    // two chunks per lane (grid-stride): 8192^2 E4M3 31.0 us with a grid of 4096 workgroups, 29.4 us with 16384
    const unsigned grid = (unsigned)std::min<int64_t>((nchunks + 2 * WWG - 1) / (2 * WWG), 0x7FFFFFFFll);
    const uint8_t* p = static_cast<const uint8_t*>(payload);
    const uint8_t* s = static_cast<const uint8_t*>(scales);
    uint4* out = static_cast<uint4*>(output);
    switch (fmt) {
        case MOR_FMT_E4M3: k_mx_dequantize<FMT_E4M3><<<grid, WWG, 0, st>>>(p, s, out, nchunks); break;
        case MOR_FMT_E5M2: k_mx_dequantize<FMT_E5M2><<<grid, WWG, 0, st>>>(p, s, out, nchunks); break;
        case MOR_FMT_E2M1: k_mx_dequantize<FMT_E2M1><<<grid, WWG, 0, st>>>(p, s, out, nchunks); break;
        case MOR_FMT_E3M2: k_mx_dequantize<FMT_E3M2><<<grid, WWG, 0, st>>>(p, s, out, nchunks); break;
        default: k_mx_dequantize<FMT_E2M3><<<grid, WWG, 0, st>>>(p, s, out, nchunks); break;
    }
    return mor_check_launch("k_mx_dequantize");
}

extern "C" int mor_fake_quantize_dual(const void* input, void* output_rows, int32_t* meta_rows, void* output_cols,
                                      int32_t* meta_cols, int64_t rows, int64_t cols, int64_t mode, int64_t sf_type,
                                      void* stream) {
    if (!input || !output_rows || !output_cols) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
    if (rows <= 0 || cols <= 0 || rows % 32 || cols % 32)
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "rows and cols must be positive multiples of 32 (got %lld x %lld)", (long long)rows, (long long)cols);
    if ((reinterpret_cast<uintptr_t>(input) | reinterpret_cast<uintptr_t>(output_rows) | reinterpret_cast<uintptr_t>(output_cols)) & 15u)
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensors must be 16-byte aligned");
    if (input == output_rows || input == output_cols)
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "the outputs must not alias the input (tiles are read while others are written)");
    const int qmode = (int)(mode % 10);
    if (qmode != 2 && qmode != 3) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "mode must be 2 (E4M3) or 3 (E5M2), got %lld", (long long)mode);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int64_t tiles = ((rows + 127) / 128) * ((cols + TILE_C - 1) / TILE_C);
    if (rows > MOR_MAX_ELEMENTS / cols) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensor too large (more than 2^35 elements)");
    const uint4* in = static_cast<const uint4*>(input);
    uint4* orow = static_cast<uint4*>(output_rows);
    uint16_t* ocol = static_cast<uint16_t*>(output_cols);
    const bool e8 = (sf_type == 2);
    const unsigned grid = (unsigned)tiles;
    const DualMap mm = dual_tile_map((cols + TILE_C - 1) / TILE_C, (rows + 127) / 128);
    if (qmode == 2) {
        if (e8) k_fq_dual<FMT_E4M3, true><<<grid, WWG, 0, st>>>(in, orow, meta_rows, ocol, meta_cols, rows, cols, 1, mm);
        else k_fq_dual<FMT_E4M3, false><<<grid, WWG, 0, st>>>(in, orow, meta_rows, ocol, meta_cols, rows, cols, 1, mm);
    } else {
        if (e8) k_fq_dual<FMT_E5M2, true><<<grid, WWG, 0, st>>>(in, orow, meta_rows, ocol, meta_cols, rows, cols, 2, mm);
        else k_fq_dual<FMT_E5M2, false><<<grid, WWG, 0, st>>>(in, orow, meta_rows, ocol, meta_cols, rows, cols, 2, mm);
    }
    return mor_check_launch("k_fq_dual");
}

namespace mor {
__global__ void k_wire_zero_u64(unsigned long long* p, int n) {
    if ((int)threadIdx.x < n) p[threadIdx.x] = 0ull;
}
}  // namespace mor

extern "C" int mor_selftest_hw_wire(uint64_t* mismatches, void* stream) {
    if (!mismatches) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "mismatches is NULL");
    hipStream_t st = static_cast<hipStream_t>(stream);
    k_wire_zero_u64<<<1, 64, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches), 4);       // (a fill kernel: capturable in a HIP graph)
    const unsigned grid = (2048u * 253u + WWG - 1) / WWG;
    k_selftest_hw_fp6<FMT_E2M3><<<grid, WWG, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches));
    k_selftest_hw_fp6<FMT_E3M2><<<grid, WWG, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches));
    k_selftest_hw_fp6_decode<FMT_E2M3><<<2, WWG, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches));
    k_selftest_hw_fp6_decode<FMT_E3M2><<<2, WWG, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches));
    k_selftest_hw_fp8_decode<FMT_E4M3><<<(128 * 201 + WWG - 1) / WWG, WWG, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches));
    k_selftest_hw_fp8_decode<FMT_E5M2><<<(128 * 201 + WWG - 1) / WWG, WWG, 0, st>>>(reinterpret_cast<unsigned long long*>(mismatches));
    return mor_check_launch("k_selftest_hw_wire");
}

extern "C" int mor_selftest_hw_fp4(uint64_t* mismatches, void* stream) {
    if (!mismatches) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "mismatches is NULL");
    hipStream_t st = static_cast<hipStream_t>(stream);
    unsigned long long* m = reinterpret_cast<unsigned long long*>(mismatches);
    k_wire_zero_u64<<<1, 64, 0, st>>>(m, 2);
    k_selftest_hw_fp4<<<(8192u * 253u + WWG - 1) / WWG, WWG, 0, st>>>(m);
    k_selftest_hw_fp4_decode<<<2, WWG, 0, st>>>(m);
    return mor_check_launch("k_selftest_hw_fp4");
}
