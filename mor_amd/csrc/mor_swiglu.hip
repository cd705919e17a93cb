// Gated activation that keeps its inputs in 8 bits:
//   forward    h = g / (1 + exp(-g)) * u, and per block of 32 along a row of g and of u the E4M3 codes and the scale byte
//              of the MX wire format (scale 2^floor(log2(448 / amax)))
//   backward   from dh and the decoded g, u, with s = 1 / (1 + exp(-g)):
//              dg = dh u s (1 + g (1 - s)),  du = dh g s
// Forward reads 4 and writes 2 + 2.0625 bytes per element, backward reads 2 + 2.0625 and writes 4.  A lane owns 8
// consecutive elements of a row, a quad of lanes a block (k_swiglu_mx / k_swiglu_mx_backward); arithmetic in fp32, one
// rounding to bf16 per result (bf16 is the tensors' type), the codes' rounding is the E4M3 grid's.
// Bound by memory: 16384 x 14336 takes 306 us forward and 286 backward, 6.2 and 6.6 TB/s (a 2 GiB copy reaches 4.9, a cold one
// of 128 MiB 6.2).  Rows that cannot be read as aligned vectors go element by element, at two to three times the time: 4096 x
// 14335 195 us forward and 231 backward, x 14336 84 and 75.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mor_common.h"
#include "mor_host.h"
#include "../../include/mor_hip.h"

namespace mor {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack2(float lo, float hi) { return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi}); }

// 1 / (1 + exp(-x)); exp and the reciprocal are the one-ulp instructions, far inside bf16's half step of 2^-8 of a value.
// They give 0 for what is below 2^-126: the reciprocal is taken of a quarter of its argument, so that the product with 1/4
// keeps a subnormal result as far down as exp(-x) is finite (x > -88.8).
__device__ __forceinline__ float sigmoid(float x) {
    return 0.25f * __builtin_amdgcn_rcpf(0.25f + __builtin_amdgcn_exp2f(__builtin_fmaf(-1.44269504f, x, -2.0f)));
}

struct SwigluShape {
    int64_t rows, cols;
    uint32_t chunks;          // rows * chunks per row
    DivU32 per_row;           // 8-element chunks per row: 4 ceil(cols / 32)
};

// 8 elements from column c on of each of N rows, zeros past the end.  VEC: the rows' chunks are 16-byte aligned and whole.
// Large tensors go past the caches: inputs and gradients beyond 2^25 elements, h beyond 2^26, codes beyond 2^27, where they
// do not stay in the last-level cache until they are used.  Forward and the quantization of h after it: 4096 x 14336 127 ->
// 113 us (117 with h past the caches), 16384 x 14336 537 -> 522; backward and two quantizations: 162 -> 159 and 749 -> 722;
// of 2048 x 14336 57.7 -> 59.9 and 77 -> 83, so not there.  Codes: 16384 x 14336 forward 327 -> 307, 8192 x 14336 133 -> 153.
__device__ __forceinline__ bool beyond(const SwigluShape& sh, int log2_elements) { return ((int64_t)sh.chunks * 8) >> log2_elements != 0; }
__device__ __forceinline__ void store_codes(uint8_t* at, uint2 q, bool nt) {
    if (nt) __builtin_nontemporal_store(((uint64_t)q.y << 32) | q.x, reinterpret_cast<uint64_t*>(at));
    else *reinterpret_cast<uint2*>(at) = q;
}
template <bool VEC, int N> __device__ __forceinline__ void load8(uint4 (&v)[N], const uint16_t* const (&row)[N], int64_t c, int64_t cols, bool nt) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = make_uint4(0, 0, 0, 0);
    if constexpr (VEC) {
        if (c < cols) load16_group(v, nt, [&](int k) { return reinterpret_cast<const uint4*>(row[k] + c); });
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = c + i < cols ? row[k][c + i] : 0u;
            v[k] = make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16));
        }
    }
}
template <bool VEC> __device__ __forceinline__ void store8(uint16_t* row, int64_t c, int64_t cols, uint4 v, bool nt) {
    if constexpr (VEC) {
        if (c < cols) store16_rt(reinterpret_cast<uint4*>(row + c), v, nt);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < cols) row[c + i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
}

// codes of the lane's 8 elements and the scale byte of the quad's block
__device__ __forceinline__ uint2 encode8(uint4 v, uint32_t& scale) {
    uint32_t m = 0;
    acc_amax_pk(m, v.x); acc_amax_pk(m, v.y); acc_amax_pk(m, v.z); acc_amax_pk(m, v.w);
    const uint32_t amax = group_umax(amax_bits_of(m), 4);                    // NaN and infinity win
    if (amax >= 0x7F800000u) { scale = 255u; return make_uint2(0, 0); }
    int e8 = 0;
    if (amax != 0) {
        const Scale sc = make_scale_e8<FMT_E4M3>(u2f(amax));
        e8 = sc.fast ? sc.e8 : (int)((f2u(Fmt<FMT_E4M3>::fmax / u2f(amax)) >> 23) & 0xFF) - 127;
        e8 = min(max(e8, -127), 127);
    }
    scale = (uint32_t)(127 - e8);
    auto pair = [&](uint32_t w) { return hw_pack2<FMT_E4M3>(ldexpf(bf16_lo(w), e8), ldexpf(bf16_hi(w), e8)) & 0xFFFFu; };
    return make_uint2(pair(v.x) | (pair(v.y) << 16), pair(v.z) | (pair(v.w) << 16));
}
__device__ __forceinline__ void decode8(uint2 q, uint32_t scale, float (&x)[8]) {
    const int de = (int)scale - 127;
    x[0] = hw_unpack<FMT_E4M3, 0>(q.x); x[1] = hw_unpack<FMT_E4M3, 1>(q.x); x[2] = hw_unpack<FMT_E4M3, 2>(q.x); x[3] = hw_unpack<FMT_E4M3, 3>(q.x);
    x[4] = hw_unpack<FMT_E4M3, 0>(q.y); x[5] = hw_unpack<FMT_E4M3, 1>(q.y); x[6] = hw_unpack<FMT_E4M3, 2>(q.y); x[7] = hw_unpack<FMT_E4M3, 3>(q.y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = scale == 255u ? u2f(0x7FC00000u) : ldexpf(x[i], de);
}

__device__ __forceinline__ uint32_t swiglu2(uint32_t g, uint32_t u) {
    const float a = bf16_lo(g), b = bf16_hi(g);
    return pack2(a * sigmoid(a) * bf16_lo(u), b * sigmoid(b) * bf16_hi(u));
}

template <bool VEC, bool KEEP>
__global__ __launch_bounds__(256) void k_swiglu_mx(const uint16_t* gate, int64_t gate_stride, const uint16_t* up, int64_t up_stride, uint16_t* out,
                                                   uint8_t* gate_codes, uint8_t* gate_scales, uint8_t* up_codes, uint8_t* up_scales, SwigluShape sh) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    const bool in = i < sh.chunks;                                           // whole quads
    const uint32_t row = div_u32(in ? i : 0u, sh.per_row);
    const int64_t c = in ? (int64_t)(i - row * sh.per_row.d) * 8 : sh.cols;
    uint4 v[2];
    load8<VEC>(v, {gate + row * gate_stride, up + row * up_stride}, c, sh.cols, beyond(sh, 25));
    const uint4 g = v[0], u = v[1];
    store8<VEC>(out + row * sh.cols, c, sh.cols, make_uint4(swiglu2(g.x, u.x), swiglu2(g.y, u.y), swiglu2(g.z, u.z), swiglu2(g.w, u.w)),
                beyond(sh, 26));
    if constexpr (KEEP) {
        uint32_t sg, su;
        const uint2 qg = encode8(g, sg), qu = encode8(u, su);
        if (in) {
            store_codes(gate_codes + (int64_t)i * 8, qg, beyond(sh, 27));
            store_codes(up_codes + (int64_t)i * 8, qu, beyond(sh, 27));
            if ((i & 3u) == 0) { gate_scales[i >> 2] = (uint8_t)sg; up_scales[i >> 2] = (uint8_t)su; }
        }
    }
}

template <bool VEC>
__global__ __launch_bounds__(256) void k_swiglu_mx_backward(const uint16_t* grad, const uint8_t* gate_codes, const uint8_t* gate_scales,
                                                            const uint8_t* up_codes, const uint8_t* up_scales, uint16_t* grad_gate,
                                                            uint16_t* grad_up, SwigluShape sh) {
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    if (i >= sh.chunks) return;
    const uint32_t row = div_u32(i, sh.per_row);
    const int64_t c = (int64_t)(i - row * sh.per_row.d) * 8;
    uint4 v[1];
    load8<VEC>(v, {grad + row * sh.cols}, c, sh.cols, beyond(sh, 25));
    const uint4 d = v[0];
    float g[8], u[8];
    decode8(*reinterpret_cast<const uint2*>(gate_codes + (int64_t)i * 8), gate_scales[i >> 2], g);
    decode8(*reinterpret_cast<const uint2*>(up_codes + (int64_t)i * 8), up_scales[i >> 2], u);
    const uint32_t dw[4] = {d.x, d.y, d.z, d.w};
    uint32_t wg[4], wu[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float a[2], b[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float x = g[2 * k + e], s = sigmoid(x), dh = e ? bf16_hi(dw[k]) : bf16_lo(dw[k]);
            a[e] = dh * u[2 * k + e] * s * (1.0f + x * (1.0f - s));
            b[e] = dh * x * s;
        }
        wg[k] = pack2(a[0], a[1]);
        wu[k] = pack2(b[0], b[1]);
    }
    store8<VEC>(grad_gate + row * sh.cols, c, sh.cols, make_uint4(wg[0], wg[1], wg[2], wg[3]), beyond(sh, 25));
    store8<VEC>(grad_up + row * sh.cols, c, sh.cols, make_uint4(wu[0], wu[1], wu[2], wu[3]), beyond(sh, 25));
}

}  // namespace mor

using namespace mor;

static int swiglu_shape(int64_t rows, int64_t cols, SwigluShape& sh) {
    if (rows <= 0 || cols <= 0) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "rows and cols must be positive (got %lld x %lld)", (long long)rows, (long long)cols);
    const int64_t blocks = cdiv(cols, 32);
    const int64_t most = (1ll << 30) - 64;                                   // a grid has fewer than 2^32 threads, four to a block
    if (blocks > most || rows > most / blocks) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensor too large (more than 2^30 - 64 blocks of 32)");
    sh = SwigluShape{rows, cols, (uint32_t)(rows * blocks * 4), make_div((uint32_t)(blocks * 4))};
    return MOR_OK;
}
static bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

extern "C" int mor_swiglu_mx(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride, void* output, void* gate_codes,
                             void* gate_scales, void* up_codes, void* up_scales, int64_t rows, int64_t cols, void* stream) {
    if (!gate || !up || !output) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
    const bool keep = gate_codes || gate_scales || up_codes || up_scales;
    if (keep && !(gate_codes && gate_scales && up_codes && up_scales)) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "codes and scales: all four pointers or none");
    SwigluShape sh;
    if (int rc = swiglu_shape(rows, cols, sh)) return rc;
    if (gate_stride < cols || up_stride < cols) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "row strides must be at least cols");
    if (!aligned_to(gate, 2) || !aligned_to(up, 2) || !aligned_to(output, 2)) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensors must be 2-byte aligned");
    if (keep && !(aligned_to(gate_codes, 8) && aligned_to(up_codes, 8))) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "codes must be 8-byte aligned");
    const bool vec = cols % 8 == 0 && gate_stride % 8 == 0 && up_stride % 8 == 0 && aligned16(gate) && aligned16(up) && aligned16(output);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned grid = (unsigned)cdiv(sh.chunks, 256);
    const uint16_t *g = static_cast<const uint16_t*>(gate), *u = static_cast<const uint16_t*>(up);
    uint16_t* o = static_cast<uint16_t*>(output);
    uint8_t *gc = static_cast<uint8_t*>(gate_codes), *gs = static_cast<uint8_t*>(gate_scales), *uc = static_cast<uint8_t*>(up_codes), *us = static_cast<uint8_t*>(up_scales);
    if (vec && keep) k_swiglu_mx<true, true><<<grid, 256, 0, st>>>(g, gate_stride, u, up_stride, o, gc, gs, uc, us, sh);
    else if (vec) k_swiglu_mx<true, false><<<grid, 256, 0, st>>>(g, gate_stride, u, up_stride, o, gc, gs, uc, us, sh);
    else if (keep) k_swiglu_mx<false, true><<<grid, 256, 0, st>>>(g, gate_stride, u, up_stride, o, gc, gs, uc, us, sh);
    else k_swiglu_mx<false, false><<<grid, 256, 0, st>>>(g, gate_stride, u, up_stride, o, gc, gs, uc, us, sh);
    return mor_check_launch("k_swiglu_mx");
}

extern "C" int mor_swiglu_mx_backward(const void* grad, const void* gate_codes, const void* gate_scales, const void* up_codes, const void* up_scales,
                                      void* grad_gate, void* grad_up, int64_t rows, int64_t cols, void* stream) {
    if (!grad || !gate_codes || !gate_scales || !up_codes || !up_scales || !grad_gate || !grad_up) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
    SwigluShape sh;
    if (int rc = swiglu_shape(rows, cols, sh)) return rc;
    if (!aligned_to(grad, 2) || !aligned_to(grad_gate, 2) || !aligned_to(grad_up, 2)) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "tensors must be 2-byte aligned");
    if (!aligned_to(gate_codes, 8) || !aligned_to(up_codes, 8)) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "codes must be 8-byte aligned");
    const bool vec = cols % 8 == 0 && aligned16(grad) && aligned16(grad_gate) && aligned16(grad_up);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const unsigned grid = (unsigned)cdiv(sh.chunks, 256);
    const uint16_t* d = static_cast<const uint16_t*>(grad);
    const uint8_t *gc = static_cast<const uint8_t*>(gate_codes), *gs = static_cast<const uint8_t*>(gate_scales), *uc = static_cast<const uint8_t*>(up_codes),
                  *us = static_cast<const uint8_t*>(up_scales);
    uint16_t *dg = static_cast<uint16_t*>(grad_gate), *du = static_cast<uint16_t*>(grad_up);
    if (vec) k_swiglu_mx_backward<true><<<grid, 256, 0, st>>>(d, gc, gs, uc, us, dg, du, sh);
    else k_swiglu_mx_backward<false><<<grid, 256, 0, st>>>(d, gc, gs, uc, us, dg, du, sh);
    return mor_check_launch("k_swiglu_mx_backward");
}
