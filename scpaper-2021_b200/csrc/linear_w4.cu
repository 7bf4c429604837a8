// Linear over 4-bit weights with group scales, few tokens: y = act(x W^T + b), W = c s + m (see quant4.cuh for
// the numbers, et_b200.h for the layout).
//
// Mathematics.  Per group of input features,
//     y[t, o] = sum_g ( s_g(o) (x_t . c_o)_g + m_g(o) (sum of x_t over g) ),
// so the tensor core multiplies codes (16 output rows x 16 features, exact) by up to eight fp16 tokens, and
// scale and minimum are applied to its fp32 sums once per group.  The sums of x are made when it is staged, by the
// same instruction with ones for codes.
// Nibbles 4 bits up are taken where they are, 16 times as large, into sums of their own.
//
// A warp walks blocks of 16 rows x 128 features (1 KB and their (s, m), in lane order), copied asynchronously up to
// seven blocks ahead into a ring of its own: most of what an SM reads is then in flight at once.  The warps of a
// thread block share 1, 2 or 4 panels of 16 rows and split the features among them, adding up in shared
// memory; a block walks panels until none is left.  Activations are staged in shared memory, in chunks when
// they do not fit.  Weights do not depend on earlier kernels: the ring is filled before the wait for them.
//
// What bounds it.  8192 -> 8192, one token: 9.8 us, 35.7 MB at 3.6 TB/s - 3 us of launch, filling of the rings and
// joining of the warps, then about 5.3 TB/s.  768 -> 2304: 2.4 us, all of it latency.  Loads into registers instead of the
// rings took 13.6 us.
#include <atomic>

#include "kernels.h"
#include "quant4.cuh"

namespace et {
namespace {

constexpr int W4_WARPS = 8;
constexpr int W4_THREADS = 32 * W4_WARPS;
constexpr size_t W4_SMEM = 227 * 1024;
constexpr uint32_t W4_ONES = 0x00010001u;  // code 1, twice

struct W4Args {
    const uint8_t* codes;
    const __half* params;
    const __half* bias;
    const __half* X;
    __half* Y;
    int T, in, out, act;
    int nb, panels;
    int wp_log;        // log2 of the panels that a thread block works on at a time
    int chunk_blocks;  // of activations staged at a time: a multiple of the warps along K
};

__device__ __forceinline__ void w4_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// MP panels of 16 rows to a warp, GB groups per block of 128 features; eight tokens.
// Shared memory: activations [rows][chunk + 64 bytes], their sums [chunk groups][8], the warps' sums, the rings.
// (Activation rows lie 64 bytes apart in the banks: eight lanes - two tokens, four pieces - meet no conflict.)
template <int MP, int GB>
struct W4Smem {
    static constexpr int DEPTH = MP == 2 ? 4 : 8;  // stages of a ring, of 2 or 1 KB of codes
    static constexpr int STAGE = MP * (1024 + 64 * GB);
    static constexpr int RINGS = W4_WARPS * DEPTH * STAGE;
    static constexpr int RED = W4_WARPS * MP * 8 * 16 * 4;
    static size_t bytes(int rows, int chunk) {
        return static_cast<size_t>(rows) * (chunk * 256 + 64) + static_cast<size_t>(chunk) * GB * 8 * 4 + RED + RINGS;
    }
};

template <int MP, int GB>
__global__ void __launch_bounds__(W4_THREADS, 2) linear_w4_kernel(const W4Args a) {
    using S = W4Smem<MP, GB>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = lane >> 2, j = lane & 3;
    const int wp = 1 << a.wp_log, wk = W4_WARPS >> a.wp_log;
    const int k0 = warp >> a.wp_log, w0 = warp & (wp - 1);
    const int t0 = blockIdx.y * 8;
    const int nt_live = a.T - t0 < 8 ? a.T - t0 : 8;
    const int rows = a.T < 8 ? a.T : 8;
    const int ldx = a.chunk_blocks * 256 + 64;
    float* xsum = reinterpret_cast<float*>(smem + rows * ldx);
    float* red = xsum + a.chunk_blocks * GB * 8;
    uint8_t* ring = reinterpret_cast<uint8_t*>(red) + S::RED + warp * (S::DEPTH * S::STAGE);

    // ---- the warp's blocks, in order: k0, k0 + wk, ... of units (MP panels) w0, w0 + wp grid, ...
    const int per_unit = a.nb > k0 ? (a.nb - k0 + wk - 1) / wk : 0;
    const int units = (a.panels + MP - 1) / MP, groups = (units + wp - 1) / wp;
    int unit = blockIdx.x * wp + w0, left = per_unit;  // of the next copy: its unit, and the unit's blocks to come
    uint32_t next_slot = 0;
    const uint32_t ring32 = smem_u32(ring) + lane * 16;
    const uint8_t *src, *src_params;
    int second;  // blocks from the first panel to the second (a last panel without one: that panel again)
    auto aim = [&]() {
        const int64_t at = static_cast<int64_t>(unit) * MP * a.nb + k0;
        second = MP == 2 && unit * MP + 1 < a.panels ? a.nb : 0;
        src = a.codes + at * 1024 + lane * 16;
        src_params = reinterpret_cast<const uint8_t*>(a.params) + (at + (lane < 16 ? 0 : second)) * (64 * GB) + (lane & 15) * 16;
    };
    aim();
    auto issue = [&]() {
        if (unit < units && per_unit > 0) {
            const uint32_t dst = ring32 + next_slot;
            w4_copy16(dst, src);
            w4_copy16(dst + 512, src + 512);
            if (MP == 2) {
                w4_copy16(dst + 1024, src + second * 1024ll);
                w4_copy16(dst + 1536, src + second * 1024ll + 512);
            }
            if ((lane & 15) < 4 * GB && (MP == 2 || lane < 16))
                w4_copy16(dst + MP * 1024 - (lane < 16 ? 0 : 256 - 64 * GB), src_params);
            src += wk * 1024;
            src_params += wk * (64 * GB);
            if (--left == 0) {
                left = per_unit;
                unit += gridDim.x * wp;
                aim();
            }
            next_slot = next_slot == (S::DEPTH - 1) * S::STAGE ? 0 : next_slot + S::STAGE;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");  // (empty past the last block, so that the count stays)
    };
#pragma unroll
    for (int u = 0; u < S::DEPTH - 1; ++u) issue();

    pdl_wait();
    pdl_launch_dependents();

    int slot = 0;
    const int per_chunk = a.chunk_blocks / wk;  // of a warp
    // the lane's token; past the last, that one again (never stored)
    uint8_t* xrow = smem + (i < nt_live ? i : nt_live - 1) * ldx + j * 16;
    for (int group = blockIdx.x; group < groups; group += gridDim.x) {
        const bool live = group * wp + w0 < units;
        float acc[MP][4];
#pragma unroll
        for (int k = 0; k < MP * 4; ++k) acc[k / 4][k % 4] = 0.f;
        for (int c = 0, b0 = 0; b0 < a.nb; ++c, b0 += a.chunk_blocks) {
            // ---- stage activations and their sums over groups (once, if they fit whole)
            // With one unit at a time a warp reads no features but those of its own blocks, and stages them alone.
            if (a.nb > a.chunk_blocks || group == static_cast<int>(blockIdx.x)) {
                if (wp > 1) __syncthreads();
                else __syncwarp();
                const int blocks = a.nb - b0 < a.chunk_blocks ? a.nb - b0 : a.chunk_blocks;
                const int pieces = blocks * 16;
                const int inside = pieces < (a.in - b0 * 128) / 8 ? pieces : (a.in - b0 * 128) / 8;
                const __half* x = a.X + static_cast<int64_t>(t0) * a.in + b0 * 128;
                uint32_t to = smem_u32(smem);
                // (a warp alone: 16 pieces a block, two blocks at a time)
                const int p0 = wp > 1 ? threadIdx.x : (warp + (lane >> 4) * W4_WARPS) * 16 + (lane & 15);
                const int step = wp > 1 ? W4_THREADS : 2 * W4_WARPS * 16;
                for (int t = 0; t < nt_live; ++t, x += a.in, to += ldx) {
#pragma unroll 4
                    for (int p = p0; p < pieces; p += step) {
                        if (p < inside) w4_copy16(to + p * 16, x + p * 8);
                        else *reinterpret_cast<uint4*>(smem + t * ldx + p * 16) = make_uint4(0, 0, 0, 0);  // (past the row)
                    }
                }
                asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
                if (wp > 1) __syncthreads();
                else __syncwarp();
                for (int b = warp; b < blocks; b += W4_WARPS) {
#pragma unroll
                    for (int g = 0; g < GB; ++g) {
                        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int n = g * (4 / GB); n < (g + 1) * (4 / GB); ++n) {
                            uint4* at = reinterpret_cast<uint4*>(xrow + b * 256 + n * 64);
                            const uint4 v = *at;
                            q4::mma(d, W4_ONES, W4_ONES, W4_ONES, W4_ONES, v.x, v.y);
                            q4::mma(d, W4_ONES, W4_ONES, W4_ONES, W4_ONES, v.z, v.w);
                            // pairs 0 and 2, 1 and 3 together: the second operand's registers below
                            if (i < nt_live) *at = make_uint4(v.x, v.z, v.y, v.w);
                        }
                        if (i == 0)
                            *reinterpret_cast<float2*>(xsum + (b * GB + g) * 8 + 2 * j) = make_float2(d[0], d[1]);
                    }
                }
                if (wp > 1) __syncthreads();
                else __syncwarp();
            }
            const int it0 = c * per_chunk, it1 = it0 + per_chunk < per_unit ? it0 + per_chunk : per_unit;
            for (int it = it0; live && it < it1; ++it) {
                asm volatile("cp.async.wait_group %0;" ::"n"(S::DEPTH - 2) : "memory");
                __syncwarp();
                issue();  // into the slot that the previous block left
                const uint8_t* st = ring + slot;
                slot = slot == (S::DEPTH - 1) * S::STAGE ? 0 : slot + S::STAGE;
                uint32_t r[MP][2][4];
#pragma unroll
                for (int m = 0; m < 2 * MP; ++m) {
                    const uint4 w = *reinterpret_cast<const uint4*>(st + m * 512 + lane * 16);
                    r[m / 2][m & 1][0] = w.x, r[m / 2][m & 1][1] = w.y, r[m / 2][m & 1][2] = w.z, r[m / 2][m & 1][3] = w.w;
                }
                const int b = k0 + it * wk - b0;  // in the chunk
                const __half2* pr = reinterpret_cast<const __half2*>(st + MP * 1024) + i * GB;
#pragma unroll
                for (int g = 0; g < GB; ++g) {
                    float d0[MP][4], d1[MP][4];
#pragma unroll
                    for (int n = g * (4 / GB); n < (g + 1) * (4 / GB); ++n) {
                        const uint4 x = *reinterpret_cast<const uint4*>(xrow + b * 256 + n * 64);
#pragma unroll
                        for (int m = 0; m < MP; ++m) {
                            constexpr uint32_t ONE = q4::NIBBLES, UP = q4::NIBBLES << 4;
                            const uint32_t l0 = r[m][0][n], l1 = r[m][1][n], h0 = l0 >> 8, h1 = l1 >> 8;
                            if (n == g * (4 / GB)) {
                                q4::mma0(d0[m], l0 & ONE, l1 & ONE, h0 & ONE, h1 & ONE, x.x, x.y);
                                q4::mma0(d1[m], l0 & UP, l1 & UP, h0 & UP, h1 & UP, x.z, x.w);
                            } else {
                                q4::mma(d0[m], l0 & ONE, l1 & ONE, h0 & ONE, h1 & ONE, x.x, x.y);
                                q4::mma(d1[m], l0 & UP, l1 & UP, h0 & UP, h1 & UP, x.z, x.w);
                            }
                        }
                    }
                    const float2 xs = *reinterpret_cast<const float2*>(xsum + (b * GB + g) * 8 + 2 * j);
#pragma unroll
                    for (int m = 0; m < MP; ++m) {
                        const float2 p0 = __half22float2(pr[m * 16 * GB + g]), p1 = __half22float2(pr[m * 16 * GB + 8 * GB + g]);
                        acc[m][0] = fmaf(fmaf(d1[m][0], 0.0625f, d0[m][0]), p0.x, fmaf(xs.x, p0.y, acc[m][0]));
                        acc[m][1] = fmaf(fmaf(d1[m][1], 0.0625f, d0[m][1]), p0.x, fmaf(xs.y, p0.y, acc[m][1]));
                        acc[m][2] = fmaf(fmaf(d1[m][2], 0.0625f, d0[m][2]), p1.x, fmaf(xs.x, p1.y, acc[m][2]));
                        acc[m][3] = fmaf(fmaf(d1[m][3], 0.0625f, d0[m][3]), p1.x, fmaf(xs.y, p1.y, acc[m][3]));
                    }
                }
            }
        }

        // ---- add up the warps of a unit: [warp][panel][token][16 rows]
        if (group != static_cast<int>(blockIdx.x)) __syncthreads();  // (the units before have been read)
#pragma unroll
        for (int m = 0; m < MP; ++m) {
            float* r = red + ((warp * MP + m) * 8 + 2 * j) * 16 + i;
            r[0] = acc[m][0];
            r[16] = acc[m][1];
            r[8] = acc[m][2];
            r[24] = acc[m][3];
        }
        __syncthreads();
        const int wide_log = 4 + a.wp_log + (MP - 1);  // outputs of the group
        for (int u = threadIdx.x; u < nt_live << wide_log; u += W4_THREADS) {
            const int t = u >> wide_log, o = u - (t << wide_log);
            const int n = (group << wide_log) + o, p = o >> 4;  // panel of the group: warp p / MP, its panel p % MP
            if (n >= a.out) continue;
            float y = 0.f;
            for (int k = 0; k < wk; ++k)
                y += red[((((k << a.wp_log) + p / MP) * MP + p % MP) * 8 + t) * 16 + (o & 15)];
            y *= 0x1p24f;
            if (a.bias) y += __half2float(__ldg(a.bias + n));
            if (a.act == ET_ACT_RELU) y = fmaxf(y, 0.f);
            if (a.act == ET_ACT_GELU)
                y = y * (0.5f + 0.5f * tanhf(y * (0.035677408136300125f * y * y + 0.7978845608028654f)));
            a.Y[static_cast<int64_t>(t0 + t) * a.out + n] = __float2half_rn(y);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Sixteen lanes per (row, block of 128 features): lane 4 n + j holds word n of lane j.
template <bool PACK>
__global__ void __launch_bounds__(256)
w4_move_kernel(const __half* __restrict__ W, __half* __restrict__ dense, uint32_t* __restrict__ codes,
               uint32_t* __restrict__ params, int in, int out, int nb, int group) {
    const int64_t u = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4;
    const int l = threadIdx.x & 15, n = l >> 2, j = l & 3;
    const int64_t units = static_cast<int64_t>(out) * nb;
    const bool live = u < units;
    const int row = live ? static_cast<int>(u / nb) : 0, b = live ? static_cast<int>(u - static_cast<int64_t>(row) * nb) : 0;
    const int k = b * 128 + n * 32 + j * 8;
    const bool in_row = live && k < in;
    const int64_t block = static_cast<int64_t>(row >> 4) * nb + b;
    uint32_t* word = codes + ((block * 2 + ((row >> 3) & 1)) * 32 + (row & 7) * 4 + j) * 4 + n;
    uint32_t* pair = params + (block * 16 + (row & 15)) * (128 / group) + n * 32 / group;
    if (PACK) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (in_row) v = *reinterpret_cast<const uint4*>(W + static_cast<int64_t>(row) * in + k);
        uint32_t r = q4::range_quad(in_row ? q4::range8(v) : q4::EMPTY_RANGE);
        for (int d = 4; d < group / 8; d <<= 1) r = q4::range_join(r, __shfl_xor_sync(0xffffffffu, r, d));
        const int first = b * 128 + n * 32 / group * group;  // of the group
        const uint32_t sm = first < in ? q4::params_of(r) : 0u;
        if (live) {
            *word = in_row ? q4::codes8<true>(v, sm, q4::inverse_of(sm)) : 0u;
            if (l % (group / 8) == 0) *pair = sm;
        }
    } else if (in_row) {
        *reinterpret_cast<uint4*>(dense + static_cast<int64_t>(row) * in + k) =
            q4::values8<true>(*word, *pair);
    }
}

int check_w4(int in, int out, int group) {
    if (in <= 0 || out <= 0) return ET_ERR_INVALID_ARG;
    if (group != 32 && group != 64 && group != 128) return ET_ERR_SHAPE;
    if (in % 16 || out % 16 || in > (1 << 24) || out > (1 << 24)) return ET_ERR_SHAPE;
    return ET_OK;
}

template <int MP, int GB>
int launch_w4(W4Args a, int slots, size_t smem, cudaStream_t stream) {
    auto kern = linear_w4_kernel<MP, GB>;
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, W4_SMEM) != cudaSuccess) return ET_ERR_CUDA;
        attr_set[dev] = true;
    }
    const int tiles = (a.T + 8 - 1) / (8), unit = MP << a.wp_log;
    const int groups = (a.panels + unit - 1) / unit;
    const int wide = slots / tiles > 1 ? slots / tiles : 1;
    const dim3 grid(groups < wide ? groups : wide, tiles);
    return launch_kernel(kern, grid, dim3(W4_THREADS), smem, stream, a) == cudaSuccess ? ET_OK : ET_ERR_CUDA;
}

template <int GB>
int plan_w4(W4Args a, cudaStream_t stream) {
    const int rows = a.T < 8 ? a.T : 8;
    const int64_t tiles = (a.T + 8 - 1) / (8);
    const int sms = sm_count() > 0 ? sm_count() : 148;
    using S1 = W4Smem<1, GB>;
    using S2 = W4Smem<2, GB>;
    static_assert(S2::RINGS + S2::RED <= S1::RINGS + 2 * S1::RED, "what is left for activations");
    constexpr size_t fixed = S1::RINGS + 2 * S1::RED;
    static_assert(W4_SMEM >= 8 * (W4_WARPS * 256 + 64) + W4_WARPS * GB * 8 * 4 + fixed, "one chunk fits");
    // All activations at once where they fit, else as many blocks as do, a whole number per warp.
    a.chunk_blocks = (a.nb + W4_WARPS - 1) / W4_WARPS * W4_WARPS;
    const size_t per_block = static_cast<size_t>(rows) * 256 + GB * 8 * 4;
    if (a.chunk_blocks * per_block + rows * 64 + fixed > W4_SMEM)
        a.chunk_blocks = static_cast<int>((W4_SMEM - fixed - rows * 64) / per_block) / W4_WARPS * W4_WARPS;
    const size_t smem = S1::bytes(rows, a.chunk_blocks), smem2 = S2::bytes(rows, a.chunk_blocks);
    // The plan that leaves the least for the busiest thread block, counted in panels; of equals the one with the most
    // outputs side by side (they share staged activations, and two panels a warp its fragments and its loop).
    int best = 0, mp = 1, slots = sms;
    for (int m = 1; m <= 2; ++m)
        for (int w = 0; w <= 2; ++w) {
            const int places = ((m == 1 ? smem : smem2) <= 113 * 1024 ? 2 : 1) * sms;
            const int64_t groups = (a.panels + (m << w) - 1) / (m << w) * tiles;
            const int cost = static_cast<int>((groups + places - 1) / places) * (m << w) * (places == sms ? 1 : 2);
            if ((w == 0 && m == 1) || cost <= best) {
                best = cost;
                a.wp_log = w;
                mp = m;
                slots = places;
            }
        }
    return mp == 1 ? launch_w4<1, GB>(a, slots, smem, stream) : launch_w4<2, GB>(a, slots, smem2, stream);
}

// Whether this kernel, eight tokens at a time, is expected to be faster than expanding the weights to operand
// tiles, which costs the same for 128 tokens as for one (linear_expand.cu).  Its time is 3 us and 0.32 ns for
// each block of 16 x 128 weights and eight tokens, fitted to B200 runs; this / expanding in us: 8192 -> 8192 at 8 tokens
// 12.6 / 32.0, 32 tokens 32.7 / 32.2, 64 tokens 61.9 / 32.1; 4096 -> 1024 at 64 tokens 7.5 / 15.3, 128 tokens 14.8 / 15.4;
// 1024 -> 4096 at 32 tokens 5.2 / 7.4, 64 tokens 8.9 / 5.8; 768 -> 2304 at 64 tokens 4.7 / 4.5; 512 -> 512 at 128
// tokens 3.5 / 3.6.
int g_w4_few = -1;  // test hook: -1 = automatic, 0 = never, 1 = always
bool w4_few_pay(int T, int in, int out) {
    if (T > 65535 * 8) return false;  // (its grid)
    if (g_w4_few >= 0) return g_w4_few != 0;
    const double blocks = static_cast<double>((in + 127) / 128) * (out / 16) * ((T + 7) / 8);
    return 3.0 + 0.00032 * blocks < linear_expand_w4_us(T, in, out) || T <= 8;
}

}  // namespace
}  // namespace et

extern "C" {

#ifdef ET_TEST_HOOKS
// Test hook: the kernel for few tokens: -1 = automatic, 0 = never, 1 = always.
void et_debug_set_w4_few(int mode) { et::g_w4_few = mode; }
// Test hook: 1 when that kernel is chosen for the size.
int et_debug_w4_few_pay(int T, int in, int out) { return et::w4_few_pay(T, in, out) ? 1 : 0; }
#endif  // ET_TEST_HOOKS

int et_w4_sizes(int in, int out, int group, size_t* code_bytes, size_t* param_bytes) {
    if (!code_bytes || !param_bytes) return ET_ERR_INVALID_ARG;
    const int st = et::check_w4(in, out, group);
    if (st != ET_OK) return st;
    const size_t blocks = static_cast<size_t>(out / 16) * ((in + 127) / 128);
    *code_bytes = blocks * 1024;
    *param_bytes = blocks * 16 * (128 / group) * 4;
    return ET_OK;
}

int et_w4_pack(const et_half* W, int in, int out, int group, uint8_t* codes, et_half* params, et_stream stream) {
    if (!W || !codes || !params) return ET_ERR_INVALID_ARG;
    const int st = et::check_w4(in, out, group);
    if (st != ET_OK) return st;
    if (!et::aligned16(W) || !et::aligned16(codes) || !et::aligned16(params)) return ET_ERR_ALIGNMENT;
    const int nb = (in + 127) / 128;
    const int64_t blocks = (static_cast<int64_t>(out) * nb * 16 + 255) / 256;
    if (blocks > INT32_MAX) return ET_ERR_SHAPE;
    et::count_launch();
    et::w4_move_kernel<true><<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        reinterpret_cast<const __half*>(W), nullptr, reinterpret_cast<uint32_t*>(codes),
        reinterpret_cast<uint32_t*>(params), in, out, nb, group);
    return cudaGetLastError() == cudaSuccess ? ET_OK : ET_ERR_CUDA;
}

int et_w4_densify(const uint8_t* codes, const et_half* params, int in, int out, int group, et_half* dense,
                  et_stream stream) {
    if (!codes || !params || !dense) return ET_ERR_INVALID_ARG;
    const int st = et::check_w4(in, out, group);
    if (st != ET_OK) return st;
    if (!et::aligned16(codes) || !et::aligned16(params) || !et::aligned16(dense)) return ET_ERR_ALIGNMENT;
    const int nb = (in + 127) / 128;
    const int64_t blocks = (static_cast<int64_t>(out) * nb * 16 + 255) / 256;
    if (blocks > INT32_MAX) return ET_ERR_SHAPE;
    et::count_launch();
    et::w4_move_kernel<false><<<static_cast<unsigned>(blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        nullptr, reinterpret_cast<__half*>(dense),
        reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(codes)),
        reinterpret_cast<uint32_t*>(const_cast<et_half*>(params)), in, out, nb, group);
    return cudaGetLastError() == cudaSuccess ? ET_OK : ET_ERR_CUDA;
}

int et_linear_w4_fwd(const uint8_t* codes, const et_half* params, int group, const et_half* bias, const et_half* X,
                     et_half* Y, int T, int in, int out, int act, et_stream stream) {
    if (!codes || !params || !X || !Y || T <= 0) return ET_ERR_INVALID_ARG;
    if (act < ET_ACT_NONE || act > ET_ACT_GELU) return ET_ERR_INVALID_ARG;
    const int st = et::check_w4(in, out, group);
    if (st != ET_OK) return st;
    if (T > 65535 * 128) return ET_ERR_SHAPE;
    if (!et::aligned16(codes) || !et::aligned16(params) || !et::aligned16(X) || !et::aligned16(Y))
        return ET_ERR_ALIGNMENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!et::w4_few_pay(T, in, out))
        return et::launch_linear_expand_w4(codes, reinterpret_cast<const __half*>(params), group,
                                           reinterpret_cast<const __half*>(bias),
                                           reinterpret_cast<const __half*>(X), reinterpret_cast<__half*>(Y), T, in,
                                           out, act, s);
    et::W4Args a = {};
    a.codes = codes;
    a.params = reinterpret_cast<const __half*>(params);
    a.bias = reinterpret_cast<const __half*>(bias);
    a.X = reinterpret_cast<const __half*>(X);
    a.Y = reinterpret_cast<__half*>(Y);
    a.T = T, a.in = in, a.out = out, a.act = act;
    a.nb = (in + 127) / 128;
    a.panels = out / 16;
    if (group == 128) return et::plan_w4<1>(a, s);
    if (group == 64) return et::plan_w4<2>(a, s);
    return et::plan_w4<4>(a, s);
}

}  // extern "C"
