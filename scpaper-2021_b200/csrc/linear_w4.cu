// Linear over 4-bit weights with group scales, few tokens: y = act(x W^T + b), W = c s + m (see quant4.cuh for
// the numbers, et_b200.h for the layout).
//
// Mathematics.  Per group of input features,
//     y[t, o] = sum_g ( s_g(o) (x_t . c_o)_g + m_g(o) (sum of x_t over g) ),
// so the tensor core multiplies codes (16 output rows x 16 features, exact) by up to eight fp16 tokens, and
// scale and minimum are applied to its fp32 sums once per group.  The sums of x come from the same instruction, with
// an operand of ones in place of the codes: they arrive in the lanes that need them.
//
// A warp walks blocks of 16 rows x 128 features (1 KB, in lane order: two 16-byte loads a lane) a few blocks
// ahead in registers; the warps of a thread block share 1, 2 or 4 panels of 16 rows and split the features among
// them, adding up in shared memory.  Activations are staged there too, in chunks when they do not fit.
// Weights do not depend on earlier kernels: the first blocks are fetched before the wait for them.
#include <atomic>

#include "kernels.h"
#include "quant4.cuh"

namespace et {
namespace {

constexpr int W4_WARPS = 8;
constexpr int W4_THREADS = 32 * W4_WARPS;
// Blocks in flight per warp (32 tokens: fewer, since a chunk of activations holds that many per warp).
template <int NT>
constexpr int W4_AHEAD_OF = NT == 4 ? 2 : 4;
constexpr int W4_X_BYTES = 96 * 1024;     // staged activations at most
constexpr uint32_t W4_ONES = 0x00010001u; // code 1, twice

struct W4Args {
    const uint4* codes;
    const __half* params;
    const __half* bias;
    const __half* X;
    __half* Y;
    int T, in, out, act;
    int nb, panels;
    int wp_log;        // log2 of the panels per thread block
    int chunk_blocks;  // staged at a time; a multiple of warps along K x blocks in flight
};

__device__ __forceinline__ uint4 ld_stream(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// GB groups per block of 128 features; NT tiles of eight tokens.
template <int GB, int NT>
__global__ void __launch_bounds__(W4_THREADS, NT == 1 ? 2 : 1) linear_w4_kernel(const W4Args a) {
    constexpr int W4_AHEAD = W4_AHEAD_OF<NT>;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = lane >> 2, j = lane & 3;
    const int wp = 1 << a.wp_log, wk = W4_WARPS >> a.wp_log;
    const int panel = blockIdx.x * wp + (warp & (wp - 1)), k0 = warp >> a.wp_log;
    const bool live = panel < a.panels;
    const int mine = live && a.nb > k0 ? (a.nb - k0 + wk - 1) / wk : 0;  // blocks k0, k0 + wk, ...
    const int t0 = blockIdx.y * 8 * NT;
    const int nt_live = a.T - t0 < 8 * NT ? a.T - t0 : 8 * NT;

    uint4 w[W4_AHEAD][2];
    uint32_t sm[W4_AHEAD][2][GB];
    auto fetch = [&](int u, int it) {
        if (it >= mine) return;
        const int64_t at = static_cast<int64_t>(panel) * a.nb + k0 + it * wk;
        w[u][0] = ld_stream(a.codes + at * 64 + lane);
        w[u][1] = ld_stream(a.codes + at * 64 + 32 + lane);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t* p = reinterpret_cast<const uint32_t*>(a.params) + (at * 16 + 8 * h + i) * GB;
            if (GB == 4) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
                sm[u][h][0] = v.x, sm[u][h][GB > 1] = v.y, sm[u][h][GB > 2 ? 2 : 0] = v.z, sm[u][h][GB > 3 ? 3 : 0] = v.w;
            } else if (GB == 2) {
                const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
                sm[u][h][0] = v.x, sm[u][h][GB > 1] = v.y;
            } else {
                sm[u][h][0] = __ldg(p);
            }
        }
    };
#pragma unroll
    for (int u = 0; u < W4_AHEAD; ++u) fetch(u, u);

    pdl_wait();
    pdl_launch_dependents();

    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;

    const int per_chunk = a.chunk_blocks / wk;  // of a warp
    // rows 64 bytes apart in the banks: eight lanes of a load (two tokens, four pieces) meet no conflict
    const int ldx = a.chunk_blocks * 256 + 64;
    for (int c = 0, b0 = 0; b0 < a.nb; ++c, b0 += a.chunk_blocks) {
        if (c > 0) __syncthreads();
        const int blocks = a.nb - b0 < a.chunk_blocks ? a.nb - b0 : a.chunk_blocks;
        for (int t = warp; t < nt_live; t += W4_WARPS) {
            const __half* x = a.X + static_cast<int64_t>(t0 + t) * a.in + b0 * 128;
            const int left = a.in - b0 * 128;
            for (int p = lane; p < blocks * 16; p += 32) {
                const bool in = p * 8 < left;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem + t * ldx + p * 16)),
                             "l"(in ? x + p * 8 : a.X), "r"(in ? 16 : 0)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        const int it0 = c * per_chunk, it1 = it0 + per_chunk < mine ? it0 + per_chunk : mine;
        for (int it = it0; it < it1; it += W4_AHEAD) {
#pragma unroll
            for (int u = 0; u < W4_AHEAD; ++u) {
                if (it + u < it1) {
                    const uint8_t* xb = smem + (k0 + (it + u) * wk - b0) * 256 + j * 16;
                    const uint32_t r0[4] = {w[u][0].x, w[u][0].y, w[u][0].z, w[u][0].w};
                    const uint32_t r1[4] = {w[u][1].x, w[u][1].y, w[u][1].z, w[u][1].w};
#pragma unroll
                    for (int g = 0; g < GB; ++g) {
                        float d[NT][4], xs[NT][4];
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int k = 0; k < 4; ++k) d[t][k] = xs[t][k] = 0.f;
#pragma unroll
                        for (int n = g * (4 / GB); n < (g + 1) * (4 / GB); ++n) {
                            uint32_t A0[4], A1[4];
#pragma unroll
                            for (int p = 0; p < 4; ++p) {
                                A0[p] = (r0[n] >> (4 * p)) & q4::NIBBLES;
                                A1[p] = (r1[n] >> (4 * p)) & q4::NIBBLES;
                            }
#pragma unroll
                            for (int t = 0; t < NT; ++t) {
                                uint4 x = make_uint4(0, 0, 0, 0);
                                if (8 * t + i < nt_live)
                                    x = *reinterpret_cast<const uint4*>(xb + (8 * t + i) * ldx + n * 64);
                                q4::mma(d[t], A0[0], A1[0], A0[1], A1[1], x.x, x.y);
                                q4::mma(d[t], A0[2], A1[2], A0[3], A1[3], x.z, x.w);
                                q4::mma(xs[t], W4_ONES, W4_ONES, W4_ONES, W4_ONES, x.x, x.y);
                                q4::mma(xs[t], W4_ONES, W4_ONES, W4_ONES, W4_ONES, x.z, x.w);
                            }
                        }
                        const float2 p0 = __half22float2(*reinterpret_cast<const __half2*>(&sm[u][0][g]));
                        const float2 p1 = __half22float2(*reinterpret_cast<const __half2*>(&sm[u][1][g]));
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            acc[t][0] = fmaf(d[t][0], p0.x, fmaf(xs[t][0], p0.y, acc[t][0]));
                            acc[t][1] = fmaf(d[t][1], p0.x, fmaf(xs[t][1], p0.y, acc[t][1]));
                            acc[t][2] = fmaf(d[t][2], p1.x, fmaf(xs[t][0], p1.y, acc[t][2]));
                            acc[t][3] = fmaf(d[t][3], p1.x, fmaf(xs[t][1], p1.y, acc[t][3]));
                        }
                    }
                }
                fetch(u, it + u + W4_AHEAD);
            }
        }
    }

    // ---- add up the warps of a panel: [warp][token][16 rows]
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float* r = red + (warp * 8 * NT + 8 * t + 2 * j) * 16 + i;
        r[0] = acc[t][0];
        r[16] = acc[t][1];
        r[8] = acc[t][2];
        r[24] = acc[t][3];
    }
    __syncthreads();
    for (int u = threadIdx.x; u < nt_live * 16 * wp; u += W4_THREADS) {
        const int t = u / (16 * wp), o = u - t * (16 * wp);
        const int n = (blockIdx.x * wp) * 16 + o;
        if (n >= a.out) continue;
        float y = 0.f;
        for (int k = 0; k < wk; ++k) y += red[(((k << a.wp_log) + (o >> 4)) * 8 * NT + t) * 16 + (o & 15)];
        y *= 0x1p24f;
        if (a.bias) y += __half2float(__ldg(a.bias + n));
        if (a.act == ET_ACT_RELU) y = fmaxf(y, 0.f);
        if (a.act == ET_ACT_GELU)
            y = y * (0.5f + 0.5f * tanhf(y * (0.035677408136300125f * y * y + 0.7978845608028654f)));
        a.Y[static_cast<int64_t>(t0 + t) * a.out + n] = __float2half_rn(y);
    }
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

template <int GB, int NT>
int launch_w4(W4Args a, cudaStream_t stream) {
    auto kern = linear_w4_kernel<GB, NT>;
    const int rows = a.T < 8 * NT ? a.T : 8 * NT;
    constexpr int ahead = W4_AHEAD_OF<NT>;
    const int wk = W4_WARPS >> a.wp_log, unit = wk * ahead;
    // (16 tokens: 32 blocks a chunk, 132 KB; 32 tokens: 16 blocks, 133 KB)
    constexpr int most = W4_X_BYTES + 64 * 1024;
    static_assert(8 * NT * (W4_WARPS * ahead * 256 + 64) <= most, "one chunk fits");
    auto staged = [&](int blocks) { return static_cast<size_t>(rows) * (static_cast<size_t>(blocks) * 256 + 64); };
    a.chunk_blocks = (a.nb + unit - 1) / unit * unit;  // all of them, or as many as fit
    if (staged(a.nb) > W4_X_BYTES || staged(a.chunk_blocks) > static_cast<size_t>(most)) {
        a.chunk_blocks = (W4_X_BYTES / rows - 64) / 256 / unit * unit;
        if (a.chunk_blocks < unit) a.chunk_blocks = unit;
    }
    size_t smem = staged(a.chunk_blocks);
    const size_t red = static_cast<size_t>(W4_WARPS) * 8 * NT * 16 * 4;
    smem = smem > red ? smem : red;
    if (smem > static_cast<size_t>(most)) return ET_ERR_SHAPE;
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess)
            return ET_ERR_CUDA;
        attr_set[dev] = true;
    }
    const int wp = 1 << a.wp_log;
    const dim3 grid((a.panels + wp - 1) / wp, (a.T + 8 * NT - 1) / (8 * NT));
    return launch_kernel(kern, grid, dim3(W4_THREADS), smem, stream, a) == cudaSuccess ? ET_OK : ET_ERR_CUDA;
}

template <int GB>
int launch_w4_tokens(const W4Args& a, cudaStream_t stream) {
    if (a.T <= 8) return launch_w4<GB, 1>(a, stream);
    if (a.T <= 16) return launch_w4<GB, 2>(a, stream);
    return launch_w4<GB, 4>(a, stream);
}

int g_w4_small = -1;  // test hook: -1 = by the token count, 0 = never, 1 = always the kernel for few tokens
constexpr int W4_SMALL_T = 32;

}  // namespace
}  // namespace et

extern "C" {

#ifdef ET_TEST_HOOKS
void et_debug_set_w4_small(int mode) { et::g_w4_small = mode; }
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
    if (T > 65535 * 32) return ET_ERR_SHAPE;
    if (!et::aligned16(codes) || !et::aligned16(params) || !et::aligned16(X) || !et::aligned16(Y))
        return ET_ERR_ALIGNMENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool few = et::g_w4_small >= 0 ? et::g_w4_small != 0 : T <= et::W4_SMALL_T;
    if (!few)
        return et::launch_linear_expand_w4(codes, reinterpret_cast<const __half*>(params), group,
                                           reinterpret_cast<const __half*>(bias),
                                           reinterpret_cast<const __half*>(X), reinterpret_cast<__half*>(Y), T, in,
                                           out, act, s);
    et::W4Args a = {};
    a.codes = reinterpret_cast<const uint4*>(codes);
    a.params = reinterpret_cast<const __half*>(params);
    a.bias = reinterpret_cast<const __half*>(bias);
    a.X = reinterpret_cast<const __half*>(X);
    a.Y = reinterpret_cast<__half*>(Y);
    a.T = T, a.in = in, a.out = out, a.act = act;
    a.nb = (in + 127) / 128;
    a.panels = out / 16;
    // Panels per thread block: as many as leave a block for every SM (they share the staged activations).
    const int sms = et::sm_count() > 0 ? et::sm_count() : 148;
    a.wp_log = 0;
    while (a.wp_log < 2 && (a.panels >> (a.wp_log + 1)) >= sms) ++a.wp_log;
    if (group == 128) return et::launch_w4_tokens<1>(a, s);
    if (group == 64) return et::launch_w4_tokens<2>(a, s);
    return et::launch_w4_tokens<4>(a, s);
}

}  // extern "C"
