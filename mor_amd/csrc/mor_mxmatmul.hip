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

static int bits_of(int fmt) { return fmt == MOR_FMT_E2M1 ? 4 : 8; }
static MxPlan mx_plan(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    MxPlan q{};
    q.splits = 1;
    // Up to 32 rows of A: bound by reading B once (64 rows of A on 4096 x 4096 in E4M3: 23 us there, 14 us in tiles).  Four
    // waves share k where there are 512 workgroups and more (one row on 14336 x 4096 in E4M3: 16.0 us, with eight 19.4),
    // eight where there are fewer (4096 x 14336 in E2M1: 8.6 us, with four 9.7).  (From 2^28 columns on the grid would have
    // 2^32 threads.)
    if (m <= 32 && n < (1ll << 28)) {
        const int64_t pieces = cdiv(k, 512);                       // the loop's unit
        q.waves = (int)std::min<int64_t>(cdiv(n, 16) >= 512 ? 4 : 8, pieces);
        q.k_per_wave = (int)(cdiv(pieces, q.waves) * 512);
        return q;
    }
    const int ks = (bits_of(a_fmt) == 4 && bits_of(b_fmt) == 4) ? 256 : 128, group = 512 / ks;
    const int64_t steps = cdiv(k, ks);
    // 256 x 256 tiles where small ones would take more than one round of 512, two to a CU (2560 x 4096 x 4096 in E4M3, 160
    // large tiles: 47 us, 55 in small ones; 2048 x 4096 x 4096, 128 of them: 46 us, 36 in small ones)
    const int64_t large_m = cdiv(m, 256), large_n = cdiv(n, 256), large = large_m * large_n;
    q.tile = large > 128 ? 256 : 128;
    q.cut_m = m;
    q.cut_n = n;
    // A last round of large tiles on few CUs takes nearly as long as a full one: its columns or rows go to small tiles instead
    // (4096 x 4608 x 4096 in E4M3, 288 tiles: 96 -> 82 us, 8192 x 4608, 576: 148 -> 137 us).  Of half a round that pays only
    // after one full one (4096 x 6144, 384 tiles: 98 -> 95 us; 4096 x 14336, 896: 203 -> 209 us).
    if (q.tile == 256 && large > 256) {
        const int64_t full = large / 256 * 256, most = large < 512 ? 128 : 64, c_n = full / large_m, c_m = full / large_n;
        if (large > full && large - c_n * large_m <= most) q.cut_n = std::min(n, c_n * 256);
        else if (large > full && large - c_m * large_n <= most) q.cut_m = std::min(m, c_m * 256);
    }
    const int64_t tiles = cdiv(m, q.tile) * cdiv(n, q.tile);
    // k is split where small tiles leave CUs idle, by the smallest of 4 us + 0.6 us a step (two workgroups share a CU
    // without slowing each other: a step waits for memory) and, when split, 3 us + 8 bytes per result and part at 4 TB/s
    // (128 x 4096 x 14336 in E4M3: 106 us whole, 28 us in 8 parts)
    int64_t splits = 1;
    if (q.tile == 128) {
        double best = 1e30;
        for (int64_t s = 1; s <= std::max<int64_t>(1, std::min<int64_t>(512 / tiles, steps / (2 * group))); ++s) {
            const double us = 0.6 * (double)cdiv(steps, s) + (s > 1 ? 3.0 + (double)s * (double)m * (double)n * 2e-6 : 0.0);
            if (us < best) { best = us; splits = s; }
        }
    }
    q.steps_per_split = (int)(cdiv(cdiv(steps, splits), group) * group);
    q.splits = (int)cdiv(steps, q.steps_per_split);
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

static bool product_format(int fmt) { return fmt == MOR_FMT_E4M3 || fmt == MOR_FMT_E5M2 || fmt == MOR_FMT_E2M1; }
static bool product_shape(int64_t m, int64_t n, int64_t k) {
    // a grid has fewer than 2^32 threads: 512 to 256 x 256 results, at most 2^22 tiles long
    return m > 0 && n > 0 && k > 0 && k % 32 == 0 && k < (1ll << 23) && m < (1ll << 30) && n < (1ll << 30) && m <= MOR_MAX_ELEMENTS / n;
}

}  // namespace mor

using namespace mor;

extern "C" size_t mor_mx_matmul_workspace_bytes(int64_t m, int64_t n, int64_t k, int a_fmt, int b_fmt) {
    if (!product_shape(m, n, k) || !product_format(a_fmt) || !product_format(b_fmt)) return 0;
    return mx_workspace(mx_plan(m, n, k, a_fmt, b_fmt), m, n, k);
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
        MxPlan small = q;
        small.tile = 128;
        return launch(rest, a_fmt, b_fmt, small, st);
    }
    if (need) args.partial = static_cast<float*>(workspace);
    if (int rc = launch(args, a_fmt, b_fmt, q, st)) return rc;
    if (!need) return MOR_OK;
    k_mx_join<<<(unsigned)std::min<int64_t>(cdiv(m * n, 1024), 2048), 256, 0, st>>>(args.partial, args.out, m * n, q.splits);
    return mor_check_launch("k_mx_join");
}
