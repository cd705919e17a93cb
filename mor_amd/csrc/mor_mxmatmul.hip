// mor_mx_matmul: A [m, k] x B [n, k]^T of two tensors in the MX wire format, on the gfx950 scaled matrix instructions,
// straight from payload and scale bytes.
//
//   out[i, j] = sum over blocks b of 2^(sa[i, b] - 127) 2^(sb[j, b] - 127) * sum over the block's 32 codes of a * b
//
// V_MFMA_SCALE_F32_32X32X64_F8F6F4 takes 32 rows x 64 codes of either side and one scale byte per row and block, so a
// lane's operands are plain 16-byte pieces of the payload (lane l = 32 h + r, row r):
//   8-bit codes: columns 16 h .. 16 h + 15 and 32 + 16 h .. 32 + 16 h + 15 of the 64;
//   4-bit codes: columns 32 h .. 32 h + 31;
//   the scale of columns 32 h .. 32 h + 31 comes from lane 32 h + r.
// B's rows go in as the instruction's first operand, so that a lane ends up with consecutive columns of the output.
//   k_mx_tile    256 x 256 or 128 x 128 tiles of the output, both operands through LDS
//   k_mx_skinny  few rows of A: B's codes go from memory to the registers of the one wave that needs them
//   k_mx_join    adds the partial sums of a k_mx_tile launch whose k was split

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <type_traits>

#include "mor_common.h"
#include "mor_host.h"
#include "../../include/mor_hip.h"

namespace mor {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int F> struct Mx;                            // code width, the instruction's format code
template <> struct Mx<FMT_E4M3> { static constexpr int bits = 8, hw = 0; };
template <> struct Mx<FMT_E5M2> { static constexpr int bits = 8, hw = 1; };
template <> struct Mx<FMT_E2M1> { static constexpr int bits = 4, hw = 4; };

struct MxOperand {
    const uint8_t* payload;
    const uint8_t* scales;
    int64_t rows;
    int scale_access;              // bytes that can be read at once at every block 0, 4, 8 ... of a row: 16, 4 or 1
};
struct MxArgs {
    MxOperand a, b;
    uint16_t* out;                 // bf16 [a.rows, b.rows]
    float* partial;                // [splits, a.rows, b.rows] when k is split, else NULL
    int k;
    int tiles_m, tiles_n;
    int steps_per_split;
    bool out16;                    // rows of the output begin on 16-byte boundaries
};

// two fp32 -> packed bf16, nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}

// 16 scale bytes of a row from block `b` on (b a multiple of 16); blocks from nb on give 127
__device__ __forceinline__ uint4 scales16(const uint8_t* row, int b, int nb, int access) {
    if (access == 16) return *reinterpret_cast<const uint4*>(row + b);             // nb is a multiple of 16
    uint32_t w[4];
    if (access == 4) {                                                             // (the loads stand in no branch: all in flight at once)
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const uint32_t*>(row + min(b + 4 * i, nb - 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = b + 4 * i < nb ? w[i] : 0x7F7F7F7Fu;
    } else {
        uint32_t e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = row[min(b + i, nb - 1)];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = b + i < nb ? e[i] : 127u;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = e[4 * i] | (e[4 * i + 1] << 8) | (e[4 * i + 2] << 16) | (e[4 * i + 3] << 24);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes at any address
__device__ __forceinline__ uint4 load16_any(const uint8_t* p) {
    struct __attribute__((packed, aligned(1))) Any { uint32_t x, y, z, w; };
    const Any v = *reinterpret_cast<const Any*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
}

// 16 bytes from memory to LDS without passing through registers: lane i's piece lands at lds + 16 i.  (The compiler does
// not see the write, so it does not wait for it before unrelated LDS reads; every reader is behind wait_and_sync().)
__device__ __forceinline__ void copy16_to_lds(uint32_t lds, const uint8_t* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// a pointer that is the same in every lane, in scalar registers
__device__ __forceinline__ const uint8_t* scalar(const uint8_t* p) {
    const uint64_t x = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const uint8_t*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)x) |
                                            ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32));
}
// everything this wave has asked for is there and every wave has got here
__device__ __forceinline__ void wait_and_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Where piece c of a row lies among the row's CH 16-byte pieces in LDS.  Eight consecutive rows, read at the same c,
// cover all 128 bytes of the banks once.
template <int CH> __device__ __forceinline__ int swizzle(int row) { return CH == 8 ? (row & 7) : ((row >> 1) & 3); }

template <int V> using Int = std::integral_constant<int, V>;

template <int FA, int FB, int T>
__global__ __launch_bounds__(256, T == 256 ? 1 : 2) void k_mx_tile(const MxArgs p) {
    constexpr int BA = Mx<FA>::bits, BB = Mx<FB>::bits;
    constexpr int KS = (BA == 4 && BB == 4) ? 256 : 128;           // columns of k per step: 128 bytes of the wider operand
    constexpr int RA = KS * BA / 8, RB = KS * BB / 8;              // bytes per row and step
    constexpr int CA = RA / 16, CB = RB / 16;
    constexpr int SUB = KS / 64;                                   // matrix instructions' depths per step
    constexpr int NB = KS / 32;                                    // scale bytes per row and step
    constexpr int SS = 16 / NB;                                    // steps per fetch of 16 scale bytes
    constexpr int S = T / 64;                                      // 32 x 32 results per wave and side; waves 2 x 2
    constexpr int A_BYTES = T * RA, STAGE = T * (RA + RB);
    constexpr int JA = T * RA / 4096, JB = T * RB / 4096;          // 16-byte pieces per thread and step
    constexpr int SR = 2 * T / 256;                                // rows whose scales a thread fetches
    __shared__ __attribute__((aligned(128))) uint8_t lds[2 * STAGE + 2 * 2 * T * 16];
    uint8_t* const s_scale = lds + 2 * STAGE;                      // [2][2 T rows: A's, then B's][16]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;

    // workgroup -> tile: each XCD takes a contiguous range of the order "8 tile rows, column by column"
    const uint32_t tiles = (uint32_t)p.tiles_m * p.tiles_n;
    const uint32_t xcd = blockIdx.x & 7u, j0 = blockIdx.x >> 3, per = tiles >> 3, rest = tiles & 7u;
    const uint32_t id = xcd * per + min(xcd, rest) + j0;
    constexpr uint32_t GM = 8;
    const uint32_t band = id / (GM * p.tiles_n), first = band * GM, high = min(GM, (uint32_t)p.tiles_m - first);
    const uint32_t in_band = id - band * GM * p.tiles_n;
    const int tn = __builtin_amdgcn_readfirstlane(in_band / high), tm = __builtin_amdgcn_readfirstlane(first + in_band - tn * high);
    const int64_t m0 = (int64_t)tm * T, n0 = (int64_t)tn * T;
    const int rows_a = (int)min((int64_t)T, p.a.rows - m0), rows_b = (int)min((int64_t)T, p.b.rows - n0);

    const int step0 = blockIdx.y * p.steps_per_split;
    const int all_steps = (p.k + KS - 1) / KS, nsteps = min(p.steps_per_split, all_steps - step0);
    const int nblocks = p.k / 32;
    const int pitch_a = p.k / 8 * BA, pitch_b = p.k / 8 * BB;
    const uint8_t* const ga = p.a.payload + m0 * pitch_a;
    const uint8_t* const gb = p.b.payload + n0 * pitch_b;

    uint32_t off_a[JA], off_b[JB];
#pragma unroll
    for (int j = 0; j < JA; ++j) {
        const int i = j * 256 + tid, row = i / CA, c = (i % CA) ^ swizzle<CA>(row);
        off_a[j] = (uint32_t)min(row, rows_a - 1) * (uint32_t)pitch_a + c * 16;
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
        const int i = j * 256 + tid, row = i / CB, c = (i % CB) ^ swizzle<CB>(row);
        off_b[j] = (uint32_t)min(row, rows_b - 1) * (uint32_t)pitch_b + c * 16;
    }
    const uint32_t lds0 = lds_offset(lds) + wave * 1024;

    // step -> buffer; rows past the operand's end repeat its last one (their results are not stored), columns past k are 0
    constexpr int J = JA + JB;
    auto copy_piece = [&](const uint8_t* ba, const uint8_t* bb, int buf, int j) {
        if (j < JA) copy16_to_lds(lds0 + buf * STAGE + j * 4096, ba, off_a[j < JA ? j : 0]);
        else copy16_to_lds(lds0 + buf * STAGE + A_BYTES + (j - JA) * 4096, bb, off_b[j >= JA ? j - JA : 0]);
    };
    auto fetch = [&](int step, int buf) {
        const int s = step0 + step;
        if ((int64_t)(s + 1) * KS <= p.k) {
            const uint8_t *ba = scalar(ga + (int64_t)s * RA), *bb = scalar(gb + (int64_t)s * RB);
#pragma unroll
            for (int j = 0; j < J; ++j) copy_piece(ba, bb, buf, j);
        } else {
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const bool of_a = j < JA;
                const int i = (of_a ? j : j - JA) * 256 + tid;
                const int c = of_a ? (i % CA) ^ swizzle<CA>(i / CA) : (i % CB) ^ swizzle<CB>(i / CB);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (of_a ? s * RA + c * 16 < pitch_a : s * RB + c * 16 < pitch_b)
                    v = *reinterpret_cast<const uint4*>(of_a ? ga + (int64_t)s * RA + off_a[of_a ? j : 0] : gb + (int64_t)s * RB + off_b[of_a ? 0 : j - JA]);
                *reinterpret_cast<uint4*>(lds + buf * STAGE + (of_a ? 0 : A_BYTES) + i * 16) = v;
            }
        }
    };
    // scale bytes: 16 per row, i.e. SS steps, at a time, through registers
    const uint8_t* scale_row[SR];
    int scale_access[SR];
#pragma unroll
    for (int i = 0; i < SR; ++i) {
        const int row = i * 256 + tid;                             // of the 2 T
        const bool of_a = row < T;
        scale_row[i] = of_a ? p.a.scales + (m0 + min(row, rows_a - 1)) * nblocks : p.b.scales + (n0 + min(row - T, rows_b - 1)) * nblocks;
        scale_access[i] = of_a ? p.a.scale_access : p.b.scale_access;
    }
    uint4 held[SR];
    auto fetch_scales = [&](int group) {
#pragma unroll
        for (int i = 0; i < SR; ++i) held[i] = scales16(scale_row[i], step0 * NB + group * 16, nblocks, scale_access[i]);
    };
    auto store_scales = [&](int group) {
#pragma unroll
        for (int i = 0; i < SR; ++i) *reinterpret_cast<uint4*>(s_scale + (group & 1) * (2 * T * 16) + (i * 256 + tid) * 16) = held[i];
    };

    // this wave's quarter of the tile
    const int wm = (wave >> 1) * (T / 2), wn = (wave & 1) * (T / 2);
    v16f acc[S][S];                                                // [B's 32 rows][A's 32 rows]
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    v8i fa[2][S], fb[2][S];
    int sa[S], sb[S];
    uint2 raw_a[S], raw_b[S];

    auto read_side = [&](auto bits, auto pieces, v8i (&f)[S], const uint8_t* base, auto depth) {
        constexpr int BITS = decltype(bits)::value, CH = decltype(pieces)::value, U = decltype(depth)::value;
        const int z = swizzle<CH>(r);
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const uint8_t* row = base + (i * 32 + r) * (CH * 16);
            if constexpr (BITS == 4) {
                const int4 v = *reinterpret_cast<const int4*>(row + ((2 * U + h) ^ z) * 16);
                f[i] = v8i{v.x, v.y, v.z, v.w, 0, 0, 0, 0};
            } else {
                const int4 v = *reinterpret_cast<const int4*>(row + ((4 * U + h) ^ z) * 16);
                const int4 w = *reinterpret_cast<const int4*>(row + ((4 * U + 2 + h) ^ z) * 16);
                f[i] = v8i{v.x, v.y, v.z, v.w, w.x, w.y, w.z, w.w};
            }
        }
    };
    auto read_codes = [&](int buf, auto depth) {
        constexpr int U = decltype(depth)::value;
        read_side(Int<BA>(), Int<CA>(), fa[U & 1], lds + buf * STAGE + wm * RA, depth);
        read_side(Int<BB>(), Int<CB>(), fb[U & 1], lds + buf * STAGE + A_BYTES + wn * RB, depth);
    };
    auto read_scales = [&](int step) {
        const uint8_t* base = s_scale + ((step / SS) & 1) * (2 * T * 16) + (step % SS) * NB;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const uint8_t *at_a = base + (wm + i * 32 + r) * 16, *at_b = base + (T + wn + i * 32 + r) * 16;
            if constexpr (NB == 8) {
                raw_a[i] = *reinterpret_cast<const uint2*>(at_a);
                raw_b[i] = *reinterpret_cast<const uint2*>(at_b);
            } else {
                raw_a[i] = make_uint2(*reinterpret_cast<const uint32_t*>(at_a), 0);
                raw_b[i] = make_uint2(*reinterpret_cast<const uint32_t*>(at_b), 0);
            }
        }
    };
    // byte u of the register an instruction of depth u gets: block 2 u + h of the step
    auto take_scales = [&]() {
        const uint32_t pick = h ? 0x07050301u : 0x06040200u;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            sa[i] = (int)__builtin_amdgcn_perm(raw_a[i].y, raw_a[i].x, pick);
            sb[i] = (int)__builtin_amdgcn_perm(raw_b[i].y, raw_b[i].x, pick);
        }
    };
    // the S x S products of one depth; between(i) goes in front of the i-th
    auto multiply = [&](auto depth, auto between) {
        constexpr int U = decltype(depth)::value;
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j) {
                between(i * S + j);
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[U & 1][i], fa[U & 1][j], acc[i][j], Mx<FB>::hw, Mx<FA>::hw,
                                                                            U, sb[i], U, sa[j]);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto nothing = [](int) {};
    // keeps the products before it before it, past branches too (no instruction)
    auto pin = [&]() {
#pragma unroll
        for (int i = 0; i < S; ++i)
#pragma unroll
            for (int j = 0; j < S; ++j) {
                if constexpr (T == 256) asm volatile("" : "+a"(acc[i][j]));
                else asm volatile("" : "+v"(acc[i][j]));
            }
    };
    auto inner_depths = [&](int buf) {
        read_codes(buf, Int<1>());
        __builtin_amdgcn_sched_barrier(0);
        multiply(Int<0>(), nothing);
        if constexpr (SUB == 4) {
            read_codes(buf, Int<2>());
            __builtin_amdgcn_sched_barrier(0);
            multiply(Int<1>(), nothing);
            read_codes(buf, Int<3>());
            __builtin_amdgcn_sched_barrier(0);
            multiply(Int<2>(), nothing);
        }
    };

    // Two buffers.  The one barrier of a step stands before its last depth, whose operands are in registers by then: past
    // it the next step's codes are in LDS for every wave and the buffer of this one is free for the step after, so the
    // first reads of the next step and the copies run beside the last products.
    const int groups = (nsteps + SS - 1) / SS;
    const int whole = min(nsteps / SS, (p.k - step0 * KS) / 512);        // groups with all their 512 columns
    fetch_scales(0);
    fetch(0, 0);
    store_scales(0);
    wait_and_sync();
    if (nsteps > 1) fetch(1, 1);
    read_codes(0, Int<0>());
    read_scales(0);
    take_scales();
    int group = 0;
    const uint8_t *next_a = scalar(ga + (int64_t)(step0 + 2) * RA), *next_b = scalar(gb + (int64_t)(step0 + 2) * RB);
    for (; group + 1 < whole; ++group) {                                 // no branch in here: all that is fetched is whole
#pragma unroll
        for (int t = 0; t < SS; ++t) {
            const int buf = t & 1;
            if (t == 0) {
#pragma unroll
                for (int i = 0; i < SR; ++i) held[i] = load16_any(scale_row[i] + step0 * NB + (group + 1) * 16);
            }
            inner_depths(buf);
            if (t == SS - 1) store_scales(group + 1);
            wait_and_sync();
            read_codes(buf ^ 1, Int<0>());
            read_scales(group * SS + t + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(Int<SUB - 1>(), [&](int i) {
                constexpr int EACH = (J + S * S - 1) / (S * S);
#pragma unroll
                for (int j = i * EACH; j < (i + 1) * EACH && j < J; ++j) copy_piece(next_a, next_b, buf, j);
                __builtin_amdgcn_sched_barrier(0);
            });
            next_a += RA;
            next_b += RB;
            take_scales();
        }
    }
    for (int s = group * SS; s < nsteps; ++s) {                          // the last whole group and a ragged one
        const int buf = s & 1;
        if (s % SS == 0 && s / SS + 1 < groups) fetch_scales(s / SS + 1);
        inner_depths(buf);
        pin();
        if (s + 1 < nsteps) {
            if (s % SS == SS - 1) store_scales(s / SS + 1);
            wait_and_sync();
            if (s + 2 < nsteps) fetch(s + 2, buf);
            read_codes(buf ^ 1, Int<0>());
            read_scales(s + 1);
        }
        multiply(Int<SUB - 1>(), nothing);
        pin();
        take_scales();
    }

    // Lane (h, r) holds, of a 32 x 32 result, row m = r of the output and columns 8 q + 4 h .. + 3 for q = 0 .. 3.
    const int64_t m_wave = m0 + wm + r, n_wave = n0 + wn;
    if (p.partial) {
        float* out = p.partial + (int64_t)blockIdx.y * p.a.rows * p.b.rows;
        const bool vec = (p.b.rows & 3) == 0;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int64_t m = m_wave + j * 32;
            if (m >= p.a.rows) continue;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t n = n_wave + i * 32 + q * 8 + h * 4;
                    float* at = out + m * p.b.rows + n;
                    if (vec) {
                        if (n < p.b.rows) *reinterpret_cast<float4*>(at) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (n + e < p.b.rows) at[e] = acc[i][j][4 * q + e];
                    }
                }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const int64_t m = m_wave + j * 32;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = pack_bf16(acc[i][j][2 * e], acc[i][j][2 * e + 1]);
            if (p.out16) {
                // exchange halves between lanes (0, r) and (1, r): 8 consecutive columns, 16 bytes, in each
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const auto x = __builtin_amdgcn_permlane32_swap(w[4 * q], w[4 * q + 2], false, false);
                    const auto y = __builtin_amdgcn_permlane32_swap(w[4 * q + 1], w[4 * q + 3], false, false);
                    const int64_t n = n_wave + i * 32 + q * 16 + h * 8;
                    if (m < p.a.rows && n < p.b.rows) *reinterpret_cast<uint4*>(p.out + m * p.b.rows + n) = make_uint4(x[0], y[0], x[1], y[1]);
                }
            } else if (m < p.a.rows) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int64_t n = n_wave + i * 32 + (e >> 2) * 8 + h * 4 + (e & 3);
                    if (n < p.b.rows) p.out[m * p.b.rows + n] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                }
            }
        }
    }
}

// partial [splits][count] -> bf16, added in the order of the splits
__global__ __launch_bounds__(256) void k_mx_join(const float* partial, uint16_t* out, int64_t count, int splits) {
    const int64_t step = (int64_t)gridDim.x * 256 * 4;
    const bool vec = (count & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 7u) == 0;
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += step) {
        if (vec) {
            float4 v = *reinterpret_cast<const float4*>(partial + i);
            for (int s = 1; s < splits; ++s) {
                const float4 w = *reinterpret_cast<const float4*>(partial + s * count + i);
                v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
            }
            *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
        } else {
            for (int64_t e = i; e < min(i + 4, count); ++e) {
                float v = partial[e];
                for (int s = 1; s < splits; ++s) v += partial[s * count + e];
                out[e] = (uint16_t)pack_bf16(v, v);
            }
        }
    }
}

// Up to 16 MT rows of A.  A workgroup owns 16 rows of B (columns of the output); its waves share k, each with its own
// part, and add their sums through LDS in wave order.  Per 128 columns a wave reads 16 rows x 64 or 128 bytes of codes
// straight into the operands of V_MFMA_SCALE_F32_16X16X128 (lane l = 16 g + r, row r: 4-bit columns 32 g .., 8-bit
// columns 16 g .. and 64 + 16 g ..; scale of columns 32 g .. from lane 16 g + r).
template <int BITS> __device__ __forceinline__ v8i codes128(const uint8_t* row, int k0, int pitch, int g) {
    if constexpr (BITS == 4) {
        const int at = k0 / 2 + 16 * g;
        const bool ok = at < pitch;
        const int4 v = *reinterpret_cast<const int4*>(row + (ok ? at : 0));
        return ok ? v8i{v.x, v.y, v.z, v.w, 0, 0, 0, 0} : v8i{0, 0, 0, 0, 0, 0, 0, 0};
    } else {
        const int at = k0 + 16 * g;
        const bool ok = at < pitch, ok2 = at + 64 < pitch;
        const int4 v = *reinterpret_cast<const int4*>(row + (ok ? at : 0)), w = *reinterpret_cast<const int4*>(row + (ok2 ? at + 64 : 0));
        return v8i{ok ? v.x : 0, ok ? v.y : 0, ok ? v.z : 0, ok ? v.w : 0, ok2 ? w.x : 0, ok2 ? w.y : 0, ok2 ? w.z : 0, ok2 ? w.w : 0};
    }
}
// bytes g, 4 + g, 8 + g, 12 + g of 16 scale bytes
__device__ __forceinline__ int scales_of_lane(uint4 v, int g) {
    const uint32_t pick = 0x0C0C0400u + 0x0101u * g;                                   // byte g of either word
    const uint32_t lo = __builtin_amdgcn_perm(v.y, v.x, pick), hi = __builtin_amdgcn_perm(v.w, v.z, pick);
    return (int)(lo | (hi << 16));
}

template <int FA, int FB, int MT>
__global__ __launch_bounds__(1024) void k_mx_skinny(const MxArgs p, int k_per_wave) {
    constexpr int BA = Mx<FA>::bits, BB = Mx<FB>::bits;
    extern __shared__ __attribute__((aligned(16))) float s_sum[];                      // [waves][MT][64 lanes][4]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int pitch_a = p.k / 8 * BA, pitch_b = p.k / 8 * BB, nblocks = p.k / 32;
    const int64_t n0 = (int64_t)blockIdx.x * 16, row_b = min(n0 + r, p.b.rows - 1);
    const uint8_t* gb = p.b.payload + row_b * pitch_b;
    const uint8_t* gsb = p.b.scales + row_b * nblocks;
    const uint8_t *ga[MT], *gsa[MT];
    v4f acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t row_a = min((int64_t)(16 * i + r), p.a.rows - 1);
        ga[i] = p.a.payload + row_a * pitch_a;
        gsa[i] = p.a.scales + row_a * nblocks;
        acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int k_end = min(p.k, (wave + 1) * k_per_wave);
    for (int k0 = wave * k_per_wave; k0 < k_end; k0 += 512) {
        v8i fb[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) fb[c] = codes128<BB>(gb, k0 + 128 * c, pitch_b, g);
        const int sb = scales_of_lane(scales16(gsb, k0 / 32, nblocks, p.b.scale_access), g);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            v8i fa[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) fa[c] = codes128<BA>(ga[i], k0 + 128 * c, pitch_a, g);
            const int sa = scales_of_lane(scales16(gsa[i], k0 / 32, nblocks, p.a.scale_access), g);
            acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[0], fa[0], acc[i], Mx<FB>::hw, Mx<FA>::hw, 0, sb, 0, sa);
            acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[1], fa[1], acc[i], Mx<FB>::hw, Mx<FA>::hw, 1, sb, 1, sa);
            acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[2], fa[2], acc[i], Mx<FB>::hw, Mx<FA>::hw, 2, sb, 2, sa);
            acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[3], fa[3], acc[i], Mx<FB>::hw, Mx<FA>::hw, 3, sb, 3, sa);
        }
    }
    v4f* sums = reinterpret_cast<v4f*>(s_sum);
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[(wave * MT + i) * 64 + lane] = acc[i];
    __syncthreads();
    // lane (g, r) of part i: row 16 i + r of the output, columns n0 + 4 g .. + 3
    for (int t = threadIdx.x; t < MT * 64; t += blockDim.x) {
        v4f v = sums[t];
        for (int w = 1; w < waves; ++w) v += sums[w * MT * 64 + t];
        const int64_t m = 16 * (t >> 6) + (t & 15), n = n0 + 4 * ((t >> 4) & 3);
        if (m >= p.a.rows) continue;
        uint16_t* at = p.out + m * p.b.rows + n;
        const uint32_t lo = pack_bf16(v[0], v[1]), hi = pack_bf16(v[2], v[3]);
        if (p.out16) {
            if (n < p.b.rows) *reinterpret_cast<uint2*>(at) = make_uint2(lo, hi);
        } else {
            const uint16_t e[4] = {(uint16_t)lo, (uint16_t)(lo >> 16), (uint16_t)hi, (uint16_t)(hi >> 16)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < p.b.rows) at[j] = e[j];
        }
    }
}

// ------------------------------------------------------------------------------------------------ which kernel
struct MxPlan {
    int tile;                      // 256, 128, or 0: k_mx_skinny
    int splits, steps_per_split;   // k_mx_tile
    int waves, k_per_wave;         // k_mx_skinny
};
static int bits_of(int fmt) { return fmt == MOR_FMT_E2M1 ? 4 : 8; }
static MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    MxPlan q{};
    q.splits = 1;
    if (m <= 64) {
        const int64_t pieces = cdiv(k, 512);                       // the loop's unit
        q.waves = (int)std::min<int64_t>(8, pieces);
        q.k_per_wave = (int)(cdiv(pieces, q.waves) * 512);
        return q;
    }
    const int ks = (bits_of(a_fmt) == 4 && bits_of(b_fmt) == 4) ? 256 : 128, group = 512 / ks;      // steps per scale fetch
    const int64_t steps = cdiv(k, ks);
    q.tile = cdiv(m, 256) * cdiv(n, 256) >= 192 ? 256 : 128;
    const int64_t tiles = cdiv(m, q.tile) * cdiv(n, q.tile);
    int64_t splits = 1;
    if (q.tile == 128 && tiles < 256) splits = std::max<int64_t>(1, std::min<int64_t>(512 / tiles, steps / (2 * group)));
    q.steps_per_split = (int)(cdiv(cdiv(steps, splits), group) * group);
    q.splits = (int)cdiv(steps, q.steps_per_split);
    return q;
}

template <int FA, int FB> static int launch_matmul(const MxArgs& args, const MxPlan& q, hipStream_t st) {
    if (q.tile == 0) {
        const unsigned grid = (unsigned)cdiv(args.b.rows, 16), threads = q.waves * 64;
        const int mt = args.a.rows <= 16 ? 1 : args.a.rows <= 32 ? 2 : 4;
        const size_t lds = (size_t)q.waves * mt * 1024;
        if (mt == 1) k_mx_skinny<FA, FB, 1><<<grid, threads, lds, st>>>(args, q.k_per_wave);
        else if (mt == 2) k_mx_skinny<FA, FB, 2><<<grid, threads, lds, st>>>(args, q.k_per_wave);
        else k_mx_skinny<FA, FB, 4><<<grid, threads, lds, st>>>(args, q.k_per_wave);
        return mor_check_launch("k_mx_skinny");
    }
    const dim3 grid((unsigned)(args.tiles_m * args.tiles_n), (unsigned)q.splits);
    if (q.tile == 256) k_mx_tile<FA, FB, 256><<<grid, 256, 0, st>>>(args);
    else k_mx_tile<FA, FB, 128><<<grid, 256, 0, st>>>(args);
    if (int rc = mor_check_launch("k_mx_tile")) return rc;
    if (args.partial) {
        const int64_t count = args.a.rows * args.b.rows;
        k_mx_join<<<(unsigned)std::min<int64_t>(cdiv(count, 1024), 2048), 256, 0, st>>>(args.partial, args.out, count, q.splits);
        return mor_check_launch("k_mx_join");
    }
    return MOR_OK;
}

template <int FA> static int launch_matmul(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st) {
    switch (b_fmt) {
        case MOR_FMT_E4M3: return launch_matmul<FA, FMT_E4M3>(args, q, st);
        case MOR_FMT_E5M2: return launch_matmul<FA, FMT_E5M2>(args, q, st);
        default: return launch_matmul<FA, FMT_E2M1>(args, q, st);
    }
}

static bool product_format(int fmt) { return fmt == MOR_FMT_E4M3 || fmt == MOR_FMT_E5M2 || fmt == MOR_FMT_E2M1; }
static bool product_shape(int64_t m, int64_t n, int64_t k) {
    return m > 0 && n > 0 && k > 0 && k % 32 == 0 && k < (1ll << 23) && m < (1ll << 31) && n < (1ll << 31) && m <= MOR_MAX_ELEMENTS / n;
}

}  // namespace mor

using namespace mor;

extern "C" size_t mor_mx_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    if (!product_shape(m, n, k) || !product_format(a_fmt) || !product_format(b_fmt)) return 0;
    const MxPlan q = mx_plan(m, n, k, a_fmt, b_fmt);
    return q.splits > 1 ? (size_t)q.splits * (size_t)m * (size_t)n * sizeof(float) : 0;
}

extern "C" int mor_mx_matmul(const void* a_payload, const void* a_scales, int a_fmt, const void* b_payload, const void* b_scales, int b_fmt,
                             void* output, int64_t m, int64_t n, int64_t k, void* workspace, size_t workspace_bytes, void* stream) {
    if (!a_payload || !a_scales || !b_payload || !b_scales || !output) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
    if (!product_format(a_fmt) || !product_format(b_fmt))
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "products take the formats E4M3, E5M2 and E2M1 (got %d and %d)", a_fmt, b_fmt);
    if (!product_shape(m, n, k))
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "products need k a positive multiple of 32 below 2^23, m and n positive and below 2^31, m * n at most 2^35 (got m %lld, n %lld, k %lld)",
                        (long long)m, (long long)n, (long long)k);
    if ((reinterpret_cast<uintptr_t>(a_payload) | reinterpret_cast<uintptr_t>(b_payload)) & 15u)
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "payloads must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(output) & 1u) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "output must be 2-byte aligned");
    const MxPlan q = mx_plan(m, n, k, a_fmt, b_fmt);
    const size_t need = q.splits > 1 ? (size_t)q.splits * (size_t)m * (size_t)n * sizeof(float) : 0;
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
        return mor_fail(MOR_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
    const int64_t nblocks = k / 32;
    auto access = [&](const void* s) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(s) | (uintptr_t)nblocks;
        return (x & 15u) == 0 ? 16 : (x & 3u) == 0 ? 4 : 1;
    };
    MxArgs args{};
    args.a = {static_cast<const uint8_t*>(a_payload), static_cast<const uint8_t*>(a_scales), m, access(a_scales)};
    args.b = {static_cast<const uint8_t*>(b_payload), static_cast<const uint8_t*>(b_scales), n, access(b_scales)};
    args.out = static_cast<uint16_t*>(output);
    args.partial = need ? static_cast<float*>(workspace) : nullptr;
    args.k = (int)k;
    args.out16 = n % 8 == 0 && aligned16(output);
    args.steps_per_split = q.steps_per_split;
    if (q.tile) {
        const int64_t tm = cdiv(m, q.tile), tn = cdiv(n, q.tile);
        if (tm * tn > 0x7FFFFFFFll) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "too many tiles");
        args.tiles_m = (int)tm;
        args.tiles_n = (int)tn;
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (a_fmt) {
        case MOR_FMT_E4M3: return launch_matmul<FMT_E4M3>(args, b_fmt, q, st);
        case MOR_FMT_E5M2: return launch_matmul<FMT_E5M2>(args, b_fmt, q, st);
        default: return launch_matmul<FMT_E2M1>(args, b_fmt, q, st);
    }
}
