// mor_mx_matmul: the choice of kernel, the entry point, and the two small kernels around k_mx_tile (mor_mxmatmul.h).
#include <algorithm>

#include "mor_mxmatmul.h"
#include "../../include/mor_hip.h"

namespace mor {

// Scale bytes [rows, blocks] -> [groups of 16 blocks][rows][16], zeros past the last block.  A tile's 256 rows then have a
// group's bytes in 4 KB that lie together; as the operands have them they are 16 bytes of each of 256 lines, a fifth of all
// the lines that k_mx_tile would fetch (4096 x 4096 x 14336 E4M3: 203 us without this kernel, 195 with it).  Bound by latency:
// 5 us for 16384 + 14336 rows of k = 4096.
__global__ __launch_bounds__(256) void k_mx_scales(const MxOperand a, const MxOperand b, uint4* out_a, uint4* out_b, int nblocks, int groups) {
    const MxOperand& o = blockIdx.y ? b : a;
    uint4* out = blockIdx.y ? out_b : out_a;
    // 16 rows x 16 groups per workgroup and step: 256 bytes of each of 16 rows are read, 256 bytes of each of 16 groups written
    const int bands = (groups + 15) / 16;
    const int64_t count = ((o.rows + 15) / 16) * bands;
    for (int64_t i = blockIdx.x; i < count; i += gridDim.x) {
        const int64_t row = i / bands * 16 + (threadIdx.x & 15);
        const int g = (int)(i % bands) * 16 + (threadIdx.x >> 4);
        if (row < o.rows && g < groups) out[g * o.rows + row] = scales16<true>(o.scales + row * nblocks, g * 16, nblocks);
    }
}

// partial [splits][count] -> bf16, added in fp32 in the order of the splits, whatever order they were computed in: the
// result does not depend on the launch.  Bound by latency (3 us) at the sizes whose k is split.
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

// A grid has fewer than 2^32 threads: past that it is cut without an error.
static bool fits_a_grid(int64_t workgroups, int waves) { return workgroups < (1ll << 32) / (waves * 64); }

static int bits_of(int fmt) { return fmt == MOR_FMT_E2M1 ? 4 : 8; }

// Estimates in us, from the measurements below (operands of three calls in turn, in part from the last-level cache).
//
// Tiles of 128 or 64 and the parts that k is split into: 4 us, and a time per step that grows where two workgroups share a
// CU's copies, but no less than the operands at 5 TB/s; for a split k 3 us more and 8 bytes per result and part at 4 TB/s.
// T = 64 whole | in parts (how many), T = 128 in eight waves, T = 128 in four | in parts:
//                             E4M3                                  E4M3 x E2M1                          E2M1
//   1000 x 1000 x 1024         4.7, 7.2, 7.4                         4.4, 6.6, 6.9                        4.2, 5.2, 5.3
//   256 x 4096 x 4096         13.4 | 15.8 (2), 20.0, 22.9            11.9 | 15.2 (2), 17.4, 20.4          10.6 | 14.2 (2), 14.4, 13.4
//   512 x 4096 x 4096         16.5, 20.3, 23.4 | 21.9 (2)            14.2, 17.7, 20.8 | 21.4 (2)          11.9, 14.6, 13.8 | 20.9 (2)
//   1024 x 4096 x 4096        30.7, 22.3, 25.6                       25.8, 19.7, 22.5                     18.1, 16.3, 15.9
//   2048 x 4096 x 4096        61.2, 42.9, 34.4                       49.5, 37.7, 32.1                     34.0, 23.8, 23.1
//   64 x 4096 x 4096          12.4 | 10.0 (4), 18.9, 22.2 | 12.5     10.8 | 9.2 (4), 15.4, 18.9 | 11.7    7.7 | 8.9 (4), 10.9, 10.8 | 10.0
//   128 x 4096 x 14336        38.0 | 20.7 (4), 63.8, 74.9 | 22.9 (8) 32.9 | 17.9 (4), 54.6, 67.0 | 21.2   28.8 | 15.8 (4), 45.4, 40.4 | 16.7
//   700 x 1000 x 14336        38.8 | 30.1 (2), 63.6, 72.5 | 26.5 (7) 33.5 | 25.4 (2), 56.0, 64.8 | 25.1   29.4 | 21.5 (2), 43.3, 39.1 | 19.2 (4)
//   64 x 65536 x 4096         68.0, 74.5, 69.1                       44.9, 49.0, 40.6                     37.4, 36.0, 34.2
//   128 x 65536 x 4096        97.0, 79.5, 72.6                       80.2, 57.2, 44.4                     56.7, 40.5, 37.1
// A mixed pair is priced as an 8-bit one: its order is the same but for 64 x 65536 x 4096 (10 % lost).  Two 4-bit operands gain
// nothing from eight waves that four, whose steps have 256 columns there too, do not give.
// More tiles than run at once only where they are a single row or column: else the operands are read too often.
static double small_tiles(MxPlan& q, int64_t m, int64_t n, int64_t k, int bits_a, int bits_b, bool split) {
    const bool both4 = bits_a == 4 && bits_b == 4;
    struct Shape { int tile, waves, columns, most; double us, shared; };           // us per step, and where all `most` run
    const Shape shapes[] = {{64, 4, 256, 512, both4 ? 0.36 : 0.52, both4 ? 0.50 : 0.78}, {128, 8, 256, 256, 1.05, 1.05}, {128, 4, both4 ? 256 : 128, 512, 0.60, 0.60}};
    const double operands = ((double)m * bits_a + (double)n * bits_b) * (double)k / 8.0 / 5.0e6;
    double best = 1e30;
    for (const Shape& s : shapes) {
        const int64_t tiles = cdiv(m, s.tile) * cdiv(n, s.tile), steps = cdiv(k, s.columns), group = 512 / s.columns;
        if (both4 && s.waves == 8) continue;
        if (tiles > s.most && (std::min(m, n) > s.tile || s.waves == 8 || !fits_a_grid(tiles, s.waves))) continue;
        const int64_t most = split ? std::max<int64_t>(1, std::min<int64_t>(s.most / tiles, steps / (2 * group))) : 1;
        for (int64_t parts = 1; parts <= most; ++parts) {
            const double over = std::min(1.0, std::max(0.0, (double)(tiles * parts - 256) / 256.0));
            const double step = (s.us + over * (s.shared - s.us)) * (double)cdiv(tiles * parts, s.most);
            const double us = 4.0 + std::max(operands, step * (double)cdiv(steps, parts)) +
                              (parts > 1 ? 3.0 + (double)parts * (double)m * (double)n * 2e-6 : 0.0);
            if (us >= best) continue;
            best = us;
            q.tile = s.tile;
            q.waves = s.waves;
            q.steps_per_split = (int)(cdiv(cdiv(steps, parts), group) * group);
            q.splits = (int)cdiv(steps, q.steps_per_split);
        }
    }
    return best;
}
// k_mx_skinny: 3 us, B at 5.6 TB/s and A, which every workgroup reads, at 12.
//                                      m = 1     4       8      16    (tiles: 1 .. 16)
//   m x 14336 x 4096 E2M1               8.6     9.2    10.0    11.7    10.3 .. 10.4
//   m x 14336 x 4096 E4M3              13.6    14.6    16.0    19.0    13.6 .. 13.0
//   m x 4096 x 14336 E4M3              13.3    13.8    14.2    16.7    16.8 .. 15.1
//   m x 4096 x 4096 E4M3 x E2M1         4.0     4.4     4.8     5.5     6.3 .. 7.4
//   m x 65536 x 4096 E4M3              50.0    54.3            72.8    62.0 .. 63.1  (from memory)
static double few_rows(int64_t m, int64_t n, int64_t k, int bits_a, int bits_b) {
    return 3.0 + (double)n * bits_b * (double)k / 8.0 / 5.6e6 + (double)(cdiv(n, 16) * m) * bits_a * (double)k / 8.0 / 12e6;
}

static MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    MxPlan q{};
    q.splits = 1;
    const int bits_a = bits_of(a_fmt), bits_b = bits_of(b_fmt);
    const int64_t large_m = cdiv(m, 256), large_n = cdiv(n, 256), large = large_m * large_n;
    // Small tiles where they run in one round of 512, two to a CU (2560 x 4096 x 4096 in E4M3, 160 large tiles: 47 us, 55 in
    // small ones; 2048 x 4096 x 4096, 128 of them: 46 us, 36 in small ones), or where large ones would be half empty.
    if (large <= 128 || std::min(m, n) <= 128) {
        const double us = small_tiles(q, m, n, k, bits_a, bits_b, true);
        // Four waves share k where there are 512 workgroups and more (one row on 14336 x 4096 in E4M3: 16.0 us, with eight
        // 19.4), eight where there are fewer (4096 x 14336 in E2M1: 8.6 us, with four 9.7).
        const int64_t pieces = cdiv(k, 512);                       // the loop's unit
        const int waves = (int)std::min<int64_t>(cdiv(n, 16) >= 512 ? 4 : 8, pieces);
        if (m > 16 || !fits_a_grid(cdiv(n, 16), waves) || few_rows(m, n, k, bits_a, bits_b) >= us) return q;
        q = MxPlan{};
        q.splits = 1;
        q.waves = waves;
        q.k_per_wave = (int)(cdiv(pieces, q.waves) * 512);
        return q;
    }
    q.tile = 256;
    q.waves = bits_a == 4 && bits_b == 4 ? 8 : 4;
    q.steps_per_split = (int)(cdiv(k, 512) * (bits_a == 4 && bits_b == 4 ? 2 : 4));
    q.cut_m = m;
    q.cut_n = n;
    // A last round of large tiles on few CUs takes nearly as long as a full one: its columns or rows go to small tiles instead
    // (4096 x 4608 x 4096 in E4M3, 288 tiles: 96 -> 74 us, 8192 x 4608, 576: 148 -> 133 us).  Of half a round that pays only
    // after one full one (4096 x 6144, 384 tiles: 98 -> 93 us; 4096 x 14336, 896: 203 -> 209 us).
    if (large > 256) {
        const int64_t full = large / 256 * 256, most = large < 512 ? 128 : 64, c_n = full / large_m, c_m = full / large_n;
        if (large > full && large - c_n * large_m <= most) q.cut_n = std::min(n, c_n * 256);
        else if (large > full && large - c_m * large_n <= most) q.cut_m = std::min(m, c_m * 256);
    }
    return q;
}

// fp32 partial sums of a split k, or the scale bytes in k_mx_scales' order
static size_t mx_workspace(const MxPlan& q, int64_t m, int64_t n, int64_t k) {
    if (q.tile == 256) return (size_t)(m + n) * (size_t)cdiv(k, 512) * 16;
    return q.splits > 1 ? (size_t)q.splits * (size_t)m * (size_t)n * sizeof(float) : 0;
}

static int launch(MxArgs args, int a_fmt, int b_fmt, const MxPlan& q, hipStream_t st) {
    args.steps_per_split = q.steps_per_split;
    if (q.tile) {
        args.tiles_m = (int)cdiv(args.a.rows, q.tile);
        args.tiles_n = (int)cdiv(args.b.rows, q.tile);
    }
    return a_fmt == MOR_FMT_E4M3 ? launch_product_e4m3(args, b_fmt, q, st) : a_fmt == MOR_FMT_E5M2 ? launch_product_e5m2(args, b_fmt, q, st)
                                                                                                   : launch_product_e2m1(args, b_fmt, q, st);
}

// what a cut last round leaves: rows or columns in small tiles
static MxPlan rest_plan(const MxPlan& q, int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    MxPlan r{};
    small_tiles(r, q.cut_m < m ? m - q.cut_m : m, q.cut_n < n ? n - q.cut_n : n, k, bits_of(a_fmt), bits_of(b_fmt), false);
    return r;
}

static bool product_format(int fmt) { return fmt == MOR_FMT_E4M3 || fmt == MOR_FMT_E5M2 || fmt == MOR_FMT_E2M1; }
static bool product_shape(int64_t m, int64_t n, int64_t k) {
    // (tiles of 128 by four waves fit a grid at any such size: m or n below 2^30 in one row or column of tiles is 2^31 threads)
    return m > 0 && n > 0 && k > 0 && k % 32 == 0 && k < (1ll << 23) && m < (1ll << 30) && n < (1ll << 30) && m <= MOR_MAX_ELEMENTS / n;
}

}  // namespace mor

using namespace mor;

extern "C" size_t mor_mx_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    if (!product_shape(m, n, k) || !product_format(a_fmt) || !product_format(b_fmt)) return 0;
    return mx_workspace(mx_plan(m, n, k, a_fmt, b_fmt), m, n, k);
}

extern "C" int mor_mx_matmul_plan(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt, int64_t* plan) {
    if (!plan) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "plan is NULL");
    if (!product_shape(m, n, k) || !product_format(a_fmt) || !product_format(b_fmt)) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "no such product");
    const MxPlan q = mx_plan(m, n, k, a_fmt, b_fmt);
    auto threads = [](const MxPlan& p, int64_t rows, int64_t cols) {
        return (p.tile ? cdiv(rows, p.tile) * cdiv(cols, p.tile) : cdiv(cols, 16)) * p.waves * 64;      // along the grid's first axis
    };
    const bool large = q.tile == 256, cut = large && (q.cut_m < m || q.cut_n < n);
    plan[0] = q.tile;
    plan[1] = q.waves;
    plan[2] = q.splits;
    plan[3] = large ? q.cut_m : m;
    plan[4] = large ? q.cut_n : n;
    plan[5] = plan[6] = 0;
    plan[7] = threads(q, plan[3], plan[4]);
    if (cut) {
        const MxPlan r = rest_plan(q, m, n, k, a_fmt, b_fmt);
        plan[5] = r.tile;
        plan[6] = r.waves;
        plan[7] = std::max(plan[7], threads(r, q.cut_m < m ? m - q.cut_m : m, q.cut_n < n ? n - q.cut_n : n));
    }
    return MOR_OK;
}

extern "C" int mor_mx_matmul(const void* a_payload, const void* a_scales, int a_fmt, const void* b_payload, const void* b_scales, int b_fmt,
                             void* output, int64_t m, int64_t n, int64_t k, void* workspace, size_t workspace_bytes, void* stream) {
    if (!a_payload || !a_scales || !b_payload || !b_scales || !output) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "NULL tensor pointer");
    if (!product_format(a_fmt) || !product_format(b_fmt))
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "products take the formats E4M3, E5M2 and E2M1 (got %d and %d)", a_fmt, b_fmt);
    if (!product_shape(m, n, k))
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "products need k a positive multiple of 32 below 2^23, m and n positive and below 2^30, m * n at most 2^35 (got m %lld, n %lld, k %lld)",
                        (long long)m, (long long)n, (long long)k);
    if ((reinterpret_cast<uintptr_t>(a_payload) | reinterpret_cast<uintptr_t>(b_payload)) & 15u)
        return mor_fail(MOR_ERR_INVALID_ARGUMENT, "payloads must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(output) & 1u) return mor_fail(MOR_ERR_INVALID_ARGUMENT, "output must be 2-byte aligned");
    const MxPlan q = mx_plan(m, n, k, a_fmt, b_fmt);
    const size_t need = mx_workspace(q, m, n, k);
    if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
        return mor_fail(MOR_ERR_WORKSPACE, "workspace of %zu bytes, 16-byte aligned, needed (got %zu)", need, workspace_bytes);
    MxArgs args{};
    args.a = {static_cast<const uint8_t*>(a_payload), static_cast<const uint8_t*>(a_scales), m};
    args.b = {static_cast<const uint8_t*>(b_payload), static_cast<const uint8_t*>(b_scales), n};
    args.out = static_cast<uint16_t*>(output);
    args.out_stride = n;
    args.out16 = n % 8 == 0 && aligned16(output);
    args.k = (int)k;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q.tile == 256) {
        const int64_t cut_m = q.cut_m, cut_n = q.cut_n;            // what the large tiles take; all of it where nothing is cut
        MxArgs rest = args;
        if (cut_m < m) {
            rest.a = {args.a.payload + cut_m * (k / 8 * bits_of(a_fmt)), args.a.scales + cut_m * (k / 32), m - cut_m};
            rest.out += cut_m * n;
            args.a.rows = cut_m;
        } else if (cut_n < n) {
            rest.b = {args.b.payload + cut_n * (k / 8 * bits_of(b_fmt)), args.b.scales + cut_n * (k / 32), n - cut_n};
            rest.out += cut_n;
            args.b.rows = cut_n;
        }
        const int groups = (int)cdiv(k, 512);
        uint4 *const scales_a = static_cast<uint4*>(workspace), *const scales_b = scales_a + cut_m * groups;
        args.scales_a = reinterpret_cast<const uint8_t*>(scales_a);
        args.scales_b = reinterpret_cast<const uint8_t*>(scales_b);
        const int64_t pieces = cdiv(std::max(cut_m, cut_n), 16) * cdiv(groups, 16);
        k_mx_scales<<<dim3((unsigned)std::min<int64_t>(pieces, 8192), 2), 256, 0, st>>>(args.a, args.b, scales_a, scales_b, (int)(k / 32), groups);
        if (int rc = mor_check_launch("k_mx_scales")) return rc;
        if (int rc = launch(args, a_fmt, b_fmt, q, st)) return rc;
        if (cut_m == m && cut_n == n) return MOR_OK;
        return launch(rest, a_fmt, b_fmt, rest_plan(q, m, n, k, a_fmt, b_fmt), st);
    }
    if (need) args.partial = static_cast<float*>(workspace);
    if (int rc = launch(args, a_fmt, b_fmt, q, st)) return rc;
    if (!need) return MOR_OK;
    k_mx_join<<<(unsigned)std::min<int64_t>(cdiv(m * n, 1024), 2048), 256, 0, st>>>(args.partial, args.out, m * n, q.splits);
    return mor_check_launch("k_mx_join");
}
