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
//   k_mx_tile    tiles of 256 x 256, 128 x 128 or 64 x 64 results, both operands through LDS
//   k_mx_skinny  few rows of A: B's codes go from memory to the registers of the one wave that needs them
//   k_mx_join    adds the partial sums of a k_mx_tile launch whose k was split

#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <algorithm>
#include <type_traits>

#include "mor_common.h"
#include "mor_host.h"

namespace mor {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// A lane's share of one side of a matrix instruction, and the form the builtin takes (of 4-bit codes it reads 4 registers).
typedef int v4i __attribute__((ext_vector_type(4)));
template <int BITS> using Codes = typename std::conditional<BITS == 4, v4i, v8i>::type;
__device__ __forceinline__ v8i operand(v4i x) { return __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1); }
__device__ __forceinline__ v8i operand(v8i x) { return x; }

template <int F> struct Mx;                            // code width, the instruction's format code
template <> struct Mx<FMT_E4M3> { static constexpr int bits = 8, hw = 0; };
template <> struct Mx<FMT_E5M2> { static constexpr int bits = 8, hw = 1; };
template <> struct Mx<FMT_E2M1> { static constexpr int bits = 4, hw = 4; };

struct MxOperand {
    const uint8_t* payload;
    const uint8_t* scales;
    int64_t rows;
};
struct MxArgs {
    MxOperand a, b;
    const uint8_t *scales_a, *scales_b;      // k_mx_tile with T = 256: as k_mx_scales leaves them
    uint16_t* out;                 // bf16 [a.rows, b.rows], out_stride elements from row to row
    int64_t out_stride;
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

// 16 bytes at any address
__device__ __forceinline__ uint4 load16_any(const uint8_t* p) {
    struct __attribute__((packed, aligned(1))) Any { uint32_t x, y, z, w; };
    const Any v = *reinterpret_cast<const Any*>(p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
// 16 scale bytes of a row of nb from block b on, 0 for blocks from nb on (their codes are 0): the last 16 of the row, moved
// down.  SHORT: the row may have fewer than 16.
template <bool SHORT> __device__ __forceinline__ uint4 scales16(const uint8_t* row, int b, int nb) {
    if (SHORT && nb < 16) {
        uint32_t e[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = row[min(b + i, nb - 1)];
#pragma unroll
        for (int i = 0; i < 16; ++i) e[i] = b + i < nb ? e[i] : 0u;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = e[4 * i] | (e[4 * i + 1] << 8) | (e[4 * i + 2] << 16) | (e[4 * i + 3] << 24);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    const int at = min(b, nb - 16), down = min(b - at, 16) * 8;        // bits; the same in every lane
    const uint4 v = load16_any(row + at);
    uint64_t lo = v.x | ((uint64_t)v.y << 32), hi = v.z | ((uint64_t)v.w << 32);
    if (down >= 64) { lo = hi; hi = 0; }
    const int d = down >= 64 ? down - 64 : down;
    if (d == 64) lo = 0;
    else if (d) { lo = (lo >> d) | (hi << (64 - d)); hi >>= d; }
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

// (m0 is reserved, which the compiler remarks on at every use of these; the clobber keeps its own settings of m0 apart)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes from memory to LDS without passing through registers: lane i's piece lands at lds + 16 i.  (The compiler does
// not see the write, so it does not wait for it before unrelated LDS reads; every reader is behind wait_and_sync().)
__device__ __forceinline__ void copy16_to_lds(uint32_t lds, const uint8_t* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void copy16_to_lds(uint32_t lds, const uint8_t* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop
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

// Where piece c of a row lies among the row's CH 16-byte pieces in LDS (c ^ swizzle): 16 consecutive rows, read at the same
// c, cover the 64 banks once (FP8 8192^3: 474 -> 450 us against an order that does so for 8 rows).
template <int CH> __device__ __forceinline__ int swizzle(int row) { return CH == 16 ? (row & 15) : CH == 8 ? ((row >> 1) & 7) : ((row >> 2) & 3); }

template <int V> using Int = std::integral_constant<int, V>;
// f(Int<0>()), ..., f(Int<N - 1>())
template <int N, int I = 0, class F> __device__ __forceinline__ void unroll(F&& f) {
    if constexpr (I < N) {
        f(Int<I>());
        unroll<N, I + 1>(f);
    }
}

// T x T results per workgroup, in steps of KS columns of k in two buffers; fp32 sums in registers throughout.
//   T = 256: steps of 128 bytes of the wider operand, one workgroup per CU.  8-bit codes: four waves of 128 x 128 results,
//   256 accumulators a lane (with eight waves of 128 x 64 the operands spill or it is no faster); two 4-bit operands: eight
//   waves (16384 x 14336 x 4096: 468 us, four waves 499), since their products are twice as fast and one wave per SIMD
//   leaves them waiting.  64 bytes in four buffers are slower (8192^3 E4M3: 450 -> 497 us): 128-byte rows are whole lines.
//   T = 128, four waves: the same steps, two workgroups per CU, which cover each other's barriers.
//   T = 128, eight waves, and T = 64, two workgroups per CU: for results that do not fill the chip with larger tiles.  A step
//   waits for its copies there, so it is twice as long, 256 columns: 1024 x 4096 x 4096 E4M3 22 us against 26 in four waves
//   and short steps, 512 x 4096 x 4096 17 us (T = 64) against 23.5, 197 x 4127 x 2080 E4M3 x E2M1 9.6 against 13.4.
// Bound by power and by what a step waits for (duration, clock and busy share of the matrix units from one counter run each;
// the chip's top clock is 2.4 GHz):
//                                     quantised normal values          one constant code
//   4096 x 4096 x 14336 E4M3          169 us, 1.69 GHz, 81 % busy      141 us, 2.12 GHz, 78 %
//   8192 x 4096 x 14336 E4M3 x E2M1   312 us, 1.75 GHz, 84 %
//   16384 x 14336 x 4096 E2M1         448 us, 1.71 GHz, 60 %           378 us, 2.34 GHz, 52 %
// 8-bit codes, 2.8 PFLOP/s: a fifth of the cycles is each step's wait for its copies.  4-bit codes, 4.3 PFLOP/s: a step's 2048
// cycles of products read 196 KB of LDS and copy 64 KB in, 2030 cycles, which overlap in part.  A last round that fills half
// the CUs costs 3 %, not 12: the others clock higher.
// The sums are fp32.  The instruction adds eight neighbouring products at a time, each cut to 2^-14 of the largest one's power
// of two, which products of two 4-bit codes do not notice; of the 8-bit codes it is what the hardware has.
template <int FA, int FB, int T, int W>
__global__ __launch_bounds__(W * 64, T == 256 || W == 8 ? 1 : 2) void k_mx_tile(const MxArgs p) {
    constexpr int BA = Mx<FA>::bits, BB = Mx<FB>::bits;
    constexpr int KS = (BA == 4 && BB == 4) || T == 64 || (T == 128 && W == 8) ? 256 : 128;
    constexpr int RA = KS * BA / 8, RB = KS * BB / 8;              // bytes per row and step
    constexpr int CA = RA / 16, CB = RB / 16;
    constexpr int SUB = KS / 64;                                   // matrix instructions' depths per step
    constexpr int NB = KS / 32;                                    // scale bytes per row and step
    constexpr int SS = 16 / NB;                                    // steps per fetch of 16 scale bytes
    constexpr int NT = W * 64;                                     // threads; waves 2 x W / 2
    constexpr int SM = T / 64, SN = T / (16 * W);                  // 32 x 32 results per wave: along m, along n
    constexpr int A_BYTES = T * RA, STAGE = T * (RA + RB);
    constexpr int JA = T * RA / (16 * NT), JB = T * RB / (16 * NT);          // 16-byte pieces per thread and step
    constexpr int SR = (2 * T + NT - 1) / NT;                      // rows whose scales a thread fetches
    constexpr int SCALES = SR * NT * 16;                           // bytes of a group's scales: A's rows, B's, and repeats of the last
    constexpr int HIGH = SM * 32, WIDE = SN * 32, PITCH = WIDE * 2 + 16;    // a wave's results: rows, columns, bytes per row in LDS
    __shared__ __attribute__((aligned(128))) uint8_t lds[std::max(2 * STAGE + 2 * SCALES, W * HIGH * PITCH)];
    uint8_t* const s_scale = lds + 2 * STAGE;                      // [2][A's rows, then B's][16]

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
        const int i = j * NT + tid, row = i / CA, c = (i % CA) ^ swizzle<CA>(row);
        off_a[j] = (uint32_t)min(row, rows_a - 1) * (uint32_t)pitch_a + c * 16;
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
        const int i = j * NT + tid, row = i / CB, c = (i % CB) ^ swizzle<CB>(row);
        off_b[j] = (uint32_t)min(row, rows_b - 1) * (uint32_t)pitch_b + c * 16;
    }
    const uint32_t lds0 = lds_offset(lds) + wave * 1024;

    // step -> buffer; rows past the operand's end repeat its last one (their results are not stored), columns past k are 0
    constexpr int J = JA + JB;
    auto copy_piece = [&](const uint8_t* ba, const uint8_t* bb, int slot, int j) {
        if (j < JA) copy16_to_lds(lds0 + slot * STAGE + j * (NT * 16), ba, off_a[j < JA ? j : 0]);
        else copy16_to_lds(lds0 + slot * STAGE + A_BYTES + (j - JA) * (NT * 16), bb, off_b[j >= JA ? j - JA : 0]);
    };
    auto fetch = [&](int step, int slot) {
        const int s = step0 + step;
        if ((int64_t)(s + 1) * KS <= p.k) {
            const uint8_t *ba = scalar(ga + (int64_t)s * RA), *bb = scalar(gb + (int64_t)s * RB);
#pragma unroll
            for (int j = 0; j < J; ++j) copy_piece(ba, bb, slot, j);
        } else {
            // (four loads at a time, in no branch of their own: a load in a branch is waited for before the next is issued)
            constexpr int AT_ONCE = 4;
#pragma unroll
            for (int j0 = 0; j0 < J; j0 += AT_ONCE) {
                v4i v[AT_ONCE];
                bool in[AT_ONCE];
#pragma unroll
                for (int e = 0; e < AT_ONCE; ++e) {
                    const int j = j0 + e;
                    if (j >= J) continue;
                    const bool of_a = j < JA;
                    const int i = (of_a ? j : j - JA) * NT + tid;
                    const int c = of_a ? (i % CA) ^ swizzle<CA>(i / CA) : (i % CB) ^ swizzle<CB>(i / CB);
                    in[e] = of_a ? s * RA + c * 16 < pitch_a : s * RB + c * 16 < pitch_b;
                    const uint8_t* from = of_a ? ga + (in[e] ? (int64_t)s * RA + off_a[of_a ? j : 0] : 0) : gb + (in[e] ? (int64_t)s * RB + off_b[of_a ? 0 : j - JA] : 0);
                    v[e] = *reinterpret_cast<const v4i*>(from);
                }
#pragma unroll
                for (int e = 0; e < AT_ONCE; ++e) {
                    const int j = j0 + e;
                    if (j >= J) continue;
                    const int i = (j < JA ? j : j - JA) * NT + tid;
                    *reinterpret_cast<v4i*>(lds + slot * STAGE + (j < JA ? 0 : A_BYTES) + i * 16) = in[e] ? v[e] : v4i{0, 0, 0, 0};
                }
            }
        }
    };
    // scale bytes: 16 per row, i.e. SS steps, at a time.  T = 256: a group's lie together (k_mx_scales) and are copied like
    // the codes; smaller tiles: straight from the operands, through registers
    const uint8_t* scale_row[SR];
#pragma unroll
    for (int i = 0; i < SR; ++i) {
        const int row = i * NT + tid;                             // of the 2 T
        const bool of_a = row < T;
        const int64_t at = of_a ? m0 + min(row, rows_a - 1) : n0 + min(row - T, rows_b - 1);
        if constexpr (T == 256) scale_row[i] = (of_a ? p.scales_a : p.scales_b) + at * 16;
        else scale_row[i] = (of_a ? p.a.scales : p.b.scales) + at * nblocks;
    }
    uint4 held[SR];
    const uint32_t scales0 = lds_offset(s_scale) + wave * 1024;
    const int64_t stride_a = p.a.rows * 16, stride_b = p.b.rows * 16;
    auto fetch_scales = [&](int group, auto whole) {
        if constexpr (T == 256) {
            const int g = step0 / SS + group;
#pragma unroll
            for (int i = 0; i < SR; ++i)
                copy16_to_lds(scales0 + (group & 1) * SCALES + i * (NT * 16), scale_row[i] + g * (i * NT + wave * 64 < T ? stride_a : stride_b));
        } else {
            const int b = step0 * NB + group * 16;
#pragma unroll
            for (int i = 0; i < SR; ++i)
                held[i] = decltype(whole)::value ? load16_any(scale_row[i] + b) : scales16<true>(scale_row[i], b, nblocks);
        }
    };
    auto store_scales = [&](int group) {
        if constexpr (T != 256) {
#pragma unroll
            for (int i = 0; i < SR; ++i) *reinterpret_cast<uint4*>(s_scale + (group & 1) * SCALES + (i * NT + tid) * 16) = held[i];
        }
    };

    // this wave's part of the tile
    const int wm = (wave / (W / 2)) * (32 * SM), wn = (wave % (W / 2)) * (32 * SN);
    v16f acc[SN][SM];                                                // [B's 32 rows][A's 32 rows]
#pragma unroll
    for (int i = 0; i < SN; ++i)
#pragma unroll
        for (int j = 0; j < SM; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    Codes<BA> fa[2][SM];                                           // the operands of two depths, used in turn
    Codes<BB> fb[2][SN];
    int sa[SM], sb[SN];
    uint2 raw_a[SM], raw_b[SN];

    // One 16-byte read of the operands of depth u of the step in a slot: the reads of a depth are issued between the products
    // of the one before it, in the order in which its own products need them (B's first rows, A's, the rest of B's).
    constexpr int PA = BA == 8 ? 2 : 1, PB = BB == 8 ? 2 : 1;      // reads per 32 rows
    constexpr int READS = SM * PA + SN * PB;
    auto read_one = [&](auto pieces, auto& f, const uint8_t* base, int i, int u, int half) {
        constexpr int CH = decltype(pieces)::value;
        constexpr bool FOUR = sizeof(f) == 16;
        const int c = FOUR ? 2 * u + h : 4 * u + 2 * half + h;
        const v4i v = *reinterpret_cast<const v4i*>(base + (i * 32 + r) * (CH * 16) + (c ^ swizzle<CH>(r)) * 16);
        if constexpr (FOUR) f = v;
        else if (half == 0) f.lo = v;
        else f.hi = v;
    };
    auto read_piece = [&](int slot, int u, int n) {
        const uint8_t *base_a = lds + slot * STAGE + wm * RA, *base_b = lds + slot * STAGE + A_BYTES + wn * RB;
        if (n < PB) read_one(Int<CB>(), fb[u & 1][0], base_b, 0, u, n);
        else if (n < PB + SM * PA) read_one(Int<CA>(), fa[u & 1][(n - PB) / PA], base_a, (n - PB) / PA, u, (n - PB) % PA);
        else read_one(Int<CB>(), fb[u & 1][(n - SM * PA) / PB], base_b, (n - SM * PA) / PB, u, (n - SM * PA) % PB);
    };
    auto read_codes = [&](int slot, int u) {
#pragma unroll
        for (int n = 0; n < READS; ++n) read_piece(slot, u, n);
    };
    auto spread_reads = [&](int slot, int u, int product) {
        constexpr int SLOTS = SM * SN > SM ? SM * SN - SM : 1, EACH = (READS + SLOTS - 1) / SLOTS;
#pragma unroll
        for (int n = product * EACH; n < (product + 1) * EACH && n < READS; ++n) read_piece(slot, u, n);
    };
    auto read_scales = [&](int step) {
        const uint8_t* base = s_scale + ((step / SS) & 1) * SCALES + (step % SS) * NB;
        auto read = [&](const uint8_t* at) {
            if constexpr (NB == 8) return *reinterpret_cast<const uint2*>(at);
            else return make_uint2(*reinterpret_cast<const uint32_t*>(at), 0);
        };
#pragma unroll
        for (int i = 0; i < SM; ++i) raw_a[i] = read(base + (wm + i * 32 + r) * 16);
#pragma unroll
        for (int i = 0; i < SN; ++i) raw_b[i] = read(base + (T + wn + i * 32 + r) * 16);
    };
    // byte u of the register an instruction of depth u gets: block 2 u + h of the step
    auto take_scales = [&]() {
        const uint32_t pick = h ? 0x07050301u : 0x06040200u;
#pragma unroll
        for (int i = 0; i < SM; ++i) sa[i] = (int)__builtin_amdgcn_perm(raw_a[i].y, raw_a[i].x, pick);
#pragma unroll
        for (int i = 0; i < SN; ++i) sb[i] = (int)__builtin_amdgcn_perm(raw_b[i].y, raw_b[i].x, pick);
    };
    // the S x S products of one depth; between(i) goes in front of the i-th
    auto multiply = [&](auto depth, auto between) {
        constexpr int U = decltype(depth)::value;
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int j = 0; j < SM; ++j) {
                between(i * SM + j);
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(fb[U & 1][i]), operand(fa[U & 1][j]), acc[i][j], Mx<FB>::hw, Mx<FA>::hw,
                                                                            U, sb[i], U, sa[j]);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto nothing = [](int) {};
    // keeps the products before it before it, past branches too (no instruction)
    auto pin = [&]() {
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int j = 0; j < SM; ++j) {
                if constexpr (T == 256 && W == 4) asm volatile("" : "+a"(acc[i][j]));
                else asm volatile("" : "+v"(acc[i][j]));
            }
    };
    auto inner_depths = [&](int slot) {
        unroll<SUB - 1>([&](auto u) {
            constexpr int U = decltype(u)::value;
            multiply(u, [&](int i) { spread_reads(slot, U + 1, i); __builtin_amdgcn_sched_barrier(0); });
        });
    };

    // Two buffers.  The one barrier of a step stands before its last depth, whose operands are in registers by then: past
    // it the next step's codes are in LDS for every wave and the buffer of this one is free for the step after, so the
    // first reads of the next step and the copies run beside the last products.
    const int groups = (nsteps + SS - 1) / SS;
    const int whole = min(nsteps / SS, (p.k - step0 * KS) / 512);        // groups with all their 512 columns
    fetch_scales(0, std::false_type());
    fetch(0, 0);
    store_scales(0);
    wait_and_sync();
    if (nsteps > 1) fetch(1, 1);
    read_codes(0, 0);
    read_scales(0);
    take_scales();
    int group = 0;
    const uint8_t *next_a = scalar(ga + (int64_t)(step0 + 2) * RA), *next_b = scalar(gb + (int64_t)(step0 + 2) * RB);
    for (; group + 1 < whole; ++group) {                                 // no branch in here: all that is fetched is whole
#pragma unroll
        for (int t = 0; t < SS; ++t) {
            const int slot = t & 1;
            if (t == 0) fetch_scales(group + 1, std::true_type());
            inner_depths(slot);
            if (t == SS - 1) store_scales(group + 1);
            wait_and_sync();
            read_scales(group * SS + t + 1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(Int<SUB - 1>(), [&](int i) {
                constexpr int EACH = (J + SM * SN - 1) / (SM * SN);
                spread_reads(slot ^ 1, 0, i);
#pragma unroll
                for (int j = i * EACH; j < (i + 1) * EACH && j < J; ++j) copy_piece(next_a, next_b, slot, j);
                __builtin_amdgcn_sched_barrier(0);
            });
            next_a += RA;
            next_b += RB;
            take_scales();
        }
    }
    if (nsteps == (group + 1) * SS && whole > group) {                   // the last group, where no ragged one follows
#pragma unroll
        for (int t = 0; t < SS; ++t) {
            inner_depths(t & 1);
            if (t + 1 < SS) {
                wait_and_sync();
                read_scales(group * SS + t + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            multiply(Int<SUB - 1>(), [&](int i) {
                if (t + 1 < SS) {
                    spread_reads((t & 1) ^ 1, 0, i);
                    if (t + 2 < SS) {
                        constexpr int EACH = (J + SM * SN - 1) / (SM * SN);
#pragma unroll
                        for (int j = i * EACH; j < (i + 1) * EACH && j < J; ++j) copy_piece(next_a, next_b, t & 1, j);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            next_a += RA;
            next_b += RB;
            if (t + 1 < SS) take_scales();
        }
        ++group;
    }
    for (int s = group * SS; s < nsteps; ++s) {                          // the last whole group and a ragged one
        const int slot = s & 1;
        if (s % SS == 0 && s / SS + 1 < groups) fetch_scales(s / SS + 1, std::false_type());
        inner_depths(slot);
        pin();
        if (s + 1 < nsteps) {
            if (s % SS == SS - 1) store_scales(s / SS + 1);
            wait_and_sync();
            if (s + 2 < nsteps) fetch(s + 2, slot);
            read_codes(slot ^ 1, 0);
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
        for (int j = 0; j < SM; ++j) {
            const int64_t m = m_wave + j * 32;
            if (m >= p.a.rows) continue;
#pragma unroll
            for (int i = 0; i < SN; ++i)
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
    // Through LDS, each wave in a part of its own, so that whole rows of its quarter (256 or 128 bytes) leave at a time: as
    // the registers hold them, a store would be 16 or 32 bytes of each of 32 rows.
    wait_and_sync();
    uint8_t* const mine = lds + wave * (HIGH * PITCH);
#pragma unroll
    for (int j = 0; j < SM; ++j)
#pragma unroll
        for (int i = 0; i < SN; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<uint2*>(mine + (j * 32 + r) * PITCH + (i * 32 + q * 8 + h * 4) * 2) =
                    make_uint2(pack_bf16(acc[i][j][4 * q], acc[i][j][4 * q + 1]), pack_bf16(acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]));
    if (p.out16) {
        constexpr int LANES = WIDE / 8, ROWS = 64 / LANES;                 // lanes per row, rows per store
        const int64_t n = n_wave + (lane % LANES) * 8;
#pragma unroll
        for (int t = 0; t < HIGH / ROWS; ++t) {
            const int row = t * ROWS + lane / LANES;
            const uint4 v = *reinterpret_cast<const uint4*>(mine + row * PITCH + (lane % LANES) * 16);
            const int64_t m = m0 + wm + row;
            if (m < p.a.rows && n < p.b.rows) store16<T == 256>(reinterpret_cast<uint4*>(p.out + m * p.out_stride + n), v);
        }
    } else {
        constexpr int LANES = WIDE / 2, ROWS = 64 / LANES;
        const int64_t n = n_wave + (lane % LANES) * 2;
        for (int t = 0; t < HIGH / ROWS; ++t) {
            const int row = t * ROWS + lane / LANES;
            const uint32_t v = *reinterpret_cast<const uint32_t*>(mine + row * PITCH + (lane % LANES) * 4);
            const int64_t m = m0 + wm + row;
            uint16_t* at = p.out + m * p.out_stride + n;
            if (m < p.a.rows && n < p.b.rows) at[0] = (uint16_t)v;
            if (m < p.a.rows && n + 1 < p.b.rows) at[1] = (uint16_t)(v >> 16);
        }
    }
}

// Up to 16 rows of A.  A workgroup owns 16 rows of B (columns of the output); its waves share k, each with its own
// part, and add their sums through LDS in wave order.  Per 128 columns a wave reads 16 rows x 64 or 128 bytes of codes
// straight into the operands of V_MFMA_SCALE_F32_16X16X128 (lane l = 16 g + r, row r: 4-bit columns 32 g .., 8-bit
// columns 16 g .. and 64 + 16 g ..; scale of columns 32 g .. from lane 16 g + r).  Bound by reading B once: one row on
// 14336 x 4096 in E2M1, 31 MB, takes 8.5 us with its launch (3.7 TB/s); holding the next 512 columns in registers meanwhile
// made it 9.0 -> 10.8, non-temporal loads 9.7.
template <int BITS> __device__ __forceinline__ Codes<BITS> codes128(const uint8_t* row, int k0, int pitch, int g) {
    const v4i zero = {0, 0, 0, 0};
    const int at = (BITS == 4 ? k0 / 2 : k0) + 16 * g;
    const v4i v = *reinterpret_cast<const v4i*>(row + (at < pitch ? at : 0));
    if constexpr (BITS == 4) return at < pitch ? v : zero;
    else {
        const v4i w = *reinterpret_cast<const v4i*>(row + (at + 64 < pitch ? at + 64 : 0));
        v8i f;
        f.lo = at < pitch ? v : zero;
        f.hi = at + 64 < pitch ? w : zero;
        return f;
    }
}
// scale bytes b + g, b + 4 + g, b + 8 + g and b + 12 + g of a row of nb, 0 past its end
__device__ __forceinline__ int scales_of_lane(const uint8_t* row, int b, int nb, int g) {
    if (b + 16 <= nb) {
        const uint4 v = load16_any(row + b);
        const uint32_t pick = 0x0C0C0400u + 0x0101u * g;                               // byte g of either word
        const uint32_t lo = __builtin_amdgcn_perm(v.y, v.x, pick), hi = __builtin_amdgcn_perm(v.w, v.z, pick);
        return (int)(lo | (hi << 16));
    }
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = row[min(b + 4 * i + g, nb - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = b + 4 * i + g < nb ? e[i] : 0u;
    return (int)(e[0] | (e[1] << 8) | (e[2] << 16) | (e[3] << 24));
}

template <int FA, int FB>
__global__ __launch_bounds__(512) void k_mx_skinny(const MxArgs p, int k_per_wave) {
    constexpr int BA = Mx<FA>::bits, BB = Mx<FB>::bits;
    extern __shared__ __attribute__((aligned(16))) float s_sum[];                      // [waves][64 lanes][4]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, g = lane >> 4;
    const int pitch_a = p.k / 8 * BA, pitch_b = p.k / 8 * BB, nblocks = p.k / 32;
    const int64_t n0 = (int64_t)blockIdx.x * 16, row_b = min(n0 + r, p.b.rows - 1);
    const uint8_t* gb = p.b.payload + row_b * pitch_b;
    const uint8_t* gsb = p.b.scales + row_b * nblocks;
    const int64_t row_a = min((int64_t)r, p.a.rows - 1);
    const uint8_t* ga = p.a.payload + row_a * pitch_a;
    const uint8_t* gsa = p.a.scales + row_a * nblocks;
    v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const int k_end = min(p.k, (wave + 1) * k_per_wave);
    for (int k0 = wave * k_per_wave; k0 < k_end; k0 += 512) {
        Codes<BB> fb[4];
        Codes<BA> fa[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) fb[c] = codes128<BB>(gb, k0 + 128 * c, pitch_b, g);
        const int sb = scales_of_lane(gsb, k0 / 32, nblocks, g);
#pragma unroll
        for (int c = 0; c < 4; ++c) fa[c] = codes128<BA>(ga, k0 + 128 * c, pitch_a, g);
        const int sa = scales_of_lane(gsa, k0 / 32, nblocks, g);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(fb[0]), operand(fa[0]), acc, Mx<FB>::hw, Mx<FA>::hw, 0, sb, 0, sa);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(fb[1]), operand(fa[1]), acc, Mx<FB>::hw, Mx<FA>::hw, 1, sb, 1, sa);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(fb[2]), operand(fa[2]), acc, Mx<FB>::hw, Mx<FA>::hw, 2, sb, 2, sa);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(fb[3]), operand(fa[3]), acc, Mx<FB>::hw, Mx<FA>::hw, 3, sb, 3, sa);
    }
    v4f* sums = reinterpret_cast<v4f*>(s_sum);
    sums[wave * 64 + lane] = acc;
    __syncthreads();
    if (wave) return;
    // lane (g, r): row r of the output, columns n0 + 4 g .. + 3
    v4f v = sums[lane];
    for (int w = 1; w < waves; ++w) v += sums[w * 64 + lane];
    const int64_t m = r, n = n0 + 4 * g;
    if (m >= p.a.rows) return;
    uint16_t* at = p.out + m * p.out_stride + n;
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

// Which kernel, and how k is divided.
struct MxPlan {
    int tile;                      // k_mx_tile: 256, 128 or 64; 0: k_mx_skinny
    int waves;                     // per workgroup
    int64_t cut_m, cut_n;          // tile 256: the rows and columns it takes, the rest in smaller tiles
    int splits, steps_per_split;   // k_mx_tile
    int k_per_wave;                // k_mx_skinny
};

template <int FA, int FB> int launch_product(const MxArgs& args, const MxPlan& q, hipStream_t st) {
    if (q.tile == 0) {
        k_mx_skinny<FA, FB><<<(unsigned)cdiv(args.b.rows, 16), q.waves * 64, q.waves * 1024, st>>>(args, q.k_per_wave);
        return mor_check_launch("k_mx_skinny");
    }
    const dim3 grid((unsigned)(args.tiles_m * args.tiles_n), (unsigned)q.splits);
    constexpr bool both4 = Mx<FA>::bits == 4 && Mx<FB>::bits == 4;
    if (q.tile == 256) k_mx_tile<FA, FB, 256, both4 ? 8 : 4><<<grid, both4 ? 512 : 256, 0, st>>>(args);
    else if (q.tile == 64) k_mx_tile<FA, FB, 64, 4><<<grid, 256, 0, st>>>(args);
    else if (both4 || q.waves == 4) k_mx_tile<FA, FB, 128, 4><<<grid, 256, 0, st>>>(args);
    else if constexpr (!both4) k_mx_tile<FA, FB, 128, 8><<<grid, 512, 0, st>>>(args);
    return mor_check_launch("k_mx_tile");
}
template <int FA> int launch_product(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st) {
    switch (b_fmt) {
        case FMT_E4M3: return launch_product<FA, FMT_E4M3>(args, q, st);
        case FMT_E5M2: return launch_product<FA, FMT_E5M2>(args, q, st);
        default: return launch_product<FA, FMT_E2M1>(args, q, st);
    }
}
// one source file per format of A
int launch_product_e4m3(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st);
int launch_product_e5m2(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st);
int launch_product_e2m1(const MxArgs& args, int b_fmt, const MxPlan& q, hipStream_t st);

}  // namespace mor
