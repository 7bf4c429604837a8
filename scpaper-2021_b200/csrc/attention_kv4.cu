// Attention of new queries over a key/value cache held in 4 bits (see quant4.cuh for the numbers, et_b200.h for
// the layout).
//
// Mathematics.  With k_t = c s + m per group g of 32 features, the score of row i is
//     q_i . k_t = sum_g ( s_g(t) (q_i . c_t)_g + m_g(t) (sum of q_i over g) ),
// so the tensor core multiplies fp16 queries by codes (exact; fp32 sums) and scale and minimum are applied to
// its results.  For the second product the scale goes to the probability instead,
//     out[d in g] = ( sum_t (p_t s_g(t)) (c_t[d] - 8)  +  sum_t p_t (m_g(t) + 8 s_g(t)) ) / sum_t p_t,
// with p s split into two fp16 numbers (22 bits) and one product for each.  (Codes less 8: sums of codes of one
// sign grow with the sequence while the output shrinks, and the tensor core cuts its fp32 sums: at 32768 tokens
// that cost half of the result's own rounding again, 3.2e-4 for 2.1e-4.)  The softmax is online; its reference is
// a recent maximum, over the tokens that the row sees, of the scaled score plus the exponent of the token's largest s,
// and moves when one passes it by 6: p s < 2^6 whatever the magnitude of V, and what is hidden from a row, or
// too unlikely to count, costs it no precision.
//
// A thread block owns up to 16 query rows that share a key/value head (the heads of a group times the query
// tokens); its four warps take 32-token tiles in turn, each with a ring of asynchronous copies of its own (page
// contents land in shared memory as they are; no thread waits for another warp in the loop).  With few rows the
// sequence's tiles are dealt out to the blocks of a cluster, which join their partial results through distributed
// shared memory, or (more than 4) to blocks that leave them to a second kernel.
//
// Layout.  Both products have the cache as their 16-row operand and eight query rows as their 8-column one: a few
// rows then waste less of the tensor core and of the registers (with the rows on the 16 side, half
// empty, the accumulators took 64 registers a thread instead of 32 at 128 features; as it is, 96 and 128 features spill 12 to
// 76 bytes of loads a thread, two row tiles of 128 features 276: at 4 x 32768 tokens, 128 features, 1.3 % of the instructions).  Lane 4 i + j holds
// word j of every group of token tau(i) = (i >> 1) + 4 (i & 1) of K, and unit i of every group of tokens j, j + 4,
// j + 8, j + 12 of V: the order in which the transposed probabilities (movmatrix) lie along the second product.
//
// What bounds it: instruction issue (four warps a scheduler issue in 50 % of the cycles at 16 x 2000 tokens of 64 features,
// 57 % at 4 x 32768 of 128).  Unpacking alone takes 1.25 instructions per element and lane (a shift and
// an AND for two codes, a subtraction for V's), scales and the softmax as much again; these run for eight rows
// whether there are that many or not (one token of heads of their own: one of eight).
#include "kernels.h"
#include "kv4.h"
#include "quant4.cuh"

namespace et {
namespace {

constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int MAX_SPLITS = 64;
constexpr int JOIN_AHEAD = 16;  // partial results that the second kernel has in flight
constexpr int MIN_CHUNK = 256;  // tokens of max_len to a split at least: two tiles per warp
constexpr int MAX_CLUSTER = 4;  // splits that join through distributed shared memory
constexpr float LOG2E = 1.4426950408889634f;

struct AttArgs {
    Kv4View c;
    const __half* Q;
    __half* Z;
    const int* table;
    const int* kv_len;
    const int* q_len;
    const __half* mask;
    float* part;   // [splits][rows][32 ng] sums, then [splits][rows][2] (reference, sum of p)
    float* part_ml;
    int table_ld, batch, seq, nhead, ratio, ldq, ldz, ldm, max_len, mask_kind;
    int tiles;        // of query rows per (sequence, key/value head)
    int splits;       // blocks along the sequence
    FastDiv by_ratio;
    float scale_log2;
    int* err_word;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {  // 16, or 0: zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// NG 32-bit words at p (shared memory, 4 NG-byte aligned)
template <int NG>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[NG]) {
    if (NG == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x, w[NG > 1] = v.y, w[NG > 2 ? 2 : 0] = v.z, w[NG > 3 ? 3 : 0] = v.w;
    } else if (NG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x, w[NG > 1] = v.y;
    } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) w[g] = reinterpret_cast<const uint32_t*>(p)[g];
    }
}
// NG 16-bit units at p, two to a word
template <int NG>
__device__ __forceinline__ void lds_units(const uint8_t* p, uint32_t (&u)[(NG + 1) / 2]) {
    if (NG == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        u[0] = v.x, u[(NG + 1) / 2 - 1] = v.y;
    } else if (NG == 2) {
        u[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
        u[0] = h[0];
        if (NG == 3) {
            u[0] |= static_cast<uint32_t>(h[1]) << 16;
            u[(NG + 1) / 2 - 1] = h[2];
        }
    }
}

template <int NG, int NT>
struct Shape {
    static constexpr int TILE = 32;  // tokens of a warp's tile: one to a lane for the parameters
    static constexpr int STAGES = NG * TILE >= 128 ? 2 : 3;
    static constexpr int CODES = TILE * 16 * NG, PARAMS = TILE * 4 * NG;
    static constexpr int STAGE = 2 * (CODES + PARAMS);  // K codes, V codes, K params, V params
    static constexpr int RING = STAGES * STAGE;
    // (s, s, m, m) of K, then of V, as fp32: a token's groups, and a pad that lets eight lanes read eight tokens
    // without a bank conflict
    static constexpr int WIDE_LD = NG % 2 ? NG : NG + 1;
    static constexpr int WARP = RING + TILE * WIDE_LD * 16;
    static constexpr int TOTAL = WARPS * WARP;
};

// Thread blocks that share an SM, by registers (and, at two stages of the widest rows, shared memory).
constexpr int blocks_per_sm(int ng, int nt) { return nt == 1 || ng <= 2 ? 4 : 3; }

// Transposes an 8 x 8 matrix of fp16: lane 4 i + j holds row i, columns 2 j and 2 j + 1, before and after.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Shared memory of this block (a pointer), or of one of the cluster (an address): what join_partials reads.
__device__ __forceinline__ float2 load2(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float2 load2(uint32_t p) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(p));
    return v;
}
__device__ __forceinline__ float4 load4(uint32_t p) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(p));
    return v;
}

// Joins n <= N partial results: ml(c) gives the place of part c's (reference, sum of p), x(c) that of eight sums.
// Everything is asked for before anything is used.
template <int N, typename ML, typename X>
__device__ __forceinline__ void join_partials(int n, float (&o)[8], float& top, float& sum, ML ml, X x) {
    float2 m[N];
    float4 v[N][2];
#pragma unroll
    for (int c = 0; c < N; ++c) {
        const int from = c < n ? c : n - 1;  // (past the last that one again: not counted below)
        const auto p = x(from);
        m[c] = load2(ml(from));
        v[c][0] = load4(p);
        v[c][1] = load4(p + 16 / (sizeof(p) == 4 ? 1 : 4));
    }
    top = m[0].x;
#pragma unroll
    for (int c = 1; c < N; ++c) top = fmaxf(top, m[c].x);
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
    for (int c = 0; c < N; ++c) {
        if (m[c].x == -INFINITY || c >= n) continue;
        const float f = exp2f(m[c].x - top);
        sum = fmaf(m[c].y, f, sum);
        const float4 &u = v[c][0], &w = v[c][1];
        o[0] = fmaf(u.x, f, o[0]), o[1] = fmaf(u.y, f, o[1]), o[2] = fmaf(u.z, f, o[2]), o[3] = fmaf(u.w, f, o[3]);
        o[4] = fmaf(w.x, f, o[4]), o[5] = fmaf(w.y, f, o[5]), o[6] = fmaf(w.z, f, o[6]), o[7] = fmaf(w.w, f, o[7]);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&o)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(o[0], o[1], o[2], o[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(o[4], o[5], o[6], o[7]);
}
// Rows that saw no key are zeros.
__device__ __forceinline__ void store_z(__half* p, const float (&o)[8], float top, float sum) {
    const float inv = top == -INFINITY ? 0.f : 1.f / sum;
    uint4 z;
    z.x = pack_half2(o[0] * inv, o[1] * inv);
    z.y = pack_half2(o[2] * inv, o[3] * inv);
    z.z = pack_half2(o[4] * inv, o[5] * inv);
    z.w = pack_half2(o[6] * inv, o[7] * inv);
    *reinterpret_cast<uint4*>(p) = z;
}

// NT: tiles of eight query rows.
template <int NG, int NT>
__global__ void __launch_bounds__(THREADS, blocks_per_sm(NG, NT)) attention_kv4_kernel(const AttArgs a) {
    using S = Shape<NG, NT>;
    constexpr int D = 32 * NG, STAGES = S::STAGES, TILE = S::TILE;
    constexpr int HALVES = TILE / 16;  // 16 tokens lie in one page
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int i = lane >> 2, j = lane & 3;
    const int tau = (i >> 1) + 4 * (i & 1);
    uint8_t* ring = smem + warp * S::WARP;
    float4* wide = reinterpret_cast<float4*>(ring + S::RING);
    pdl_wait();
    pdl_launch_dependents();

    const int split = blockIdx.x;
    const int rt = blockIdx.y % a.tiles, kvh = blockIdx.y / a.tiles;
    const int b = blockIdx.z;
    const int row0 = rt * 8 * NT;  // row r is query token r / ratio, head kvh * ratio + r % ratio

    // ---- everything that waits for nothing is asked for at once: lengths, queries, page numbers
    int len = __ldcg(a.kv_len + b);
    int nq = a.q_len ? __ldcg(a.q_len + b) : a.seq;
    uint32_t qf[NG][NT][4];  // row 8 t + i: features 32 g + 8 j .. + 8
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int r = row0 + 8 * t + i, qi = a.by_ratio.div(r), head = kvh * a.ratio + r - qi * a.ratio;
        const __half* q = a.Q + (static_cast<int64_t>(b) * a.seq + qi) * a.ldq + head * a.c.dh[0] + 8 * j;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (qi < a.seq && 32 * g + 8 * j < a.c.dh[0]) v = __ldcg(reinterpret_cast<const uint4*>(q + 32 * g));
            qf[g][t][0] = v.x, qf[g][t][1] = v.y, qf[g][t][2] = v.z, qf[g][t][3] = v.w;
        }
    }
    // The warps of a sequence's blocks take its tiles in turn: shares are even whatever its length, and known before
    // it.  Page numbers: of 16 tokens to a lane, BATCH tiles at a time.  What the table holds past the sequence's end is
    // read, but neither followed nor reported.
    constexpr int BATCH = 32 / HALVES;
    const int turn = split * WARPS + warp, turns = a.splits * WARPS;  // the warp's tiles: turn, turn + turns, ...
    const int* table = a.table + static_cast<int64_t>(b) * a.table_ld;
    auto position = [&](int n) { return ((n + lane / HALVES) * turns + turn) * TILE + lane % HALVES * 16; };
    auto entry = [&](int n) {
        const int pos = position(n), e = pos >> a.c.page_shift;
        return pos < a.max_len && e < a.table_ld ? __ldcg(table + e) : -1;
    };
    int raw = entry(0), raw_next = entry(BATCH);

    if (len > a.max_len) {
        if (threadIdx.x == 0) atomicCAS(a.err_word, 0, DEV_BAD_PAGE);
        len = a.max_len;
    }
    len = len < 0 ? 0 : len;
    nq = nq < 0 ? 0 : (nq > a.seq ? a.seq : nq);
    if (row0 >= nq * a.ratio) return;  // (rows are ordered by query token)
    int end, least;  // the largest and smallest number of tokens that a row sees: the last and first row's
    {
        const int last = (row0 + 8 * NT < nq * a.ratio ? row0 + 8 * NT : nq * a.ratio) - 1;
        if (a.mask_kind == ET_MASK_CAUSAL) {
            least = len - nq + static_cast<int>(a.by_ratio.div(row0)) + 1;
            end = len - nq + static_cast<int>(a.by_ratio.div(last)) + 1;
        } else {
            least = end = len;
        }
        end = end < 0 ? 0 : end;
    }
    const int ntile = (end + TILE - 1) / TILE;
    const int mine = ntile > turn ? (ntile - turn + turns - 1) / turns : 0;
    auto checked = [&](int n, int id) {  // page of the lane's 16 tokens, or -1: nothing to read
        if (position(n) >= end || n + lane / HALVES >= mine) return -1;
        if (id >= 0 && id < a.c.num_pages) return id;
        atomicCAS(a.err_word, 0, DEV_BAD_PAGE);
        return -1;
    };
    int pages = checked(0, raw), pages_next = checked(BATCH, raw_next);
    // Copies tile n of this warp (called with n = 0, 1, 2, ... in order), zeros where nothing is to be read: per 16
    // tokens 16 NG pieces of 16 bytes of either codes and 4 NG of either parameters (K's by lanes 0 .., V's by
    // lanes 16 ..).
    const uint32_t ring32 = smem_u32(ring) + lane * 16;
    const uint8_t* code_base[2] = {a.c.codes[0] + lane * 16, a.c.codes[1] + lane * 16};
    const uint8_t* param_base = reinterpret_cast<const uint8_t*>(a.c.params[lane >> 4]) + (lane & 15) * 16;
    const uint32_t param_at = 2 * S::CODES + (lane >> 4) * (S::PARAMS - 256);
    int next_pos = turn * TILE;
    auto issue = [&](int n) {
        if (n < mine) {
            if (n != 0 && n % BATCH == 0) {
                pages = pages_next;
                pages_next = checked(n + BATCH, entry(n + BATCH));
            }
            const uint32_t st = ring32 + (n % STAGES) * S::STAGE;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int id = __shfl_sync(0xffffffffu, pages, n % BATCH * HALVES + h);
                const int have = id < 0 ? 0 : 16;
                const int64_t row = kv4_row(a.c, max(id, 0), next_pos + 16 * h, kvh);
#pragma unroll
                for (int of = 0; of < 2; ++of)
#pragma unroll
                    for (int u = 0; u < (16 * NG + 31) / 32; ++u)
                        if (u * 32 + 32 <= 16 * NG || u * 32 + lane < 16 * NG)
                            cp_async16(st + of * S::CODES + h * 256 * NG + u * 512,
                                       code_base[of] + row * (16 * NG) + u * 512, have);
                if (NG == 4 || (lane & 15) < 4 * NG)
                    cp_async16(st + param_at + h * 64 * NG, param_base + row * (4 * NG), have);
            }
        }
        next_pos += turns * TILE;
        cp_async_commit();  // (an empty group past the last tile, so that the count stays)
    };
#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) issue(n);

    // ---- the rows' queries, scaled by a power of two of their own to at most 2^11: room for the factor 16 that makes
    // up for the nibbles which K's codes are multiplied at (4 bits up, every second pair).  Lossless where the row's
    // largest is below 2^11; above, the power is 2^-1 to 2^-5, and what falls below the type's normal numbers is rounded
    // to its grid of 2^-24: by 2^-25, 2^-35 of the largest (a score's fp32 sums are off by 2^-23 of their own sizes)
    int limit[NT][2];     // tokens that rows 8 t + 2 j, 8 t + 2 j + 1 see
    uint64_t qs[NG][NT];  // rows 8 t + 2 j, + 1: sums over the group, in the units of the first product
    float unit[NT][2];    // those units times scale and log2(e)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        uint32_t big = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) big = max(big, max(qf[g][t][k] & 0x7fffu, (qf[g][t][k] >> 16) & 0x7fffu));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^k, k = 10 - exponent of the largest (0 for rows of zeros and rows that are not finite)
        const float largest = __half2float(__ushort_as_half(static_cast<unsigned short>(big)));
        const int k2 = big == 0 || big >= 0x7c00u ? 0 : 137 - static_cast<int>(__float_as_uint(largest) >> 23);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + k2) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(127 + 20 - k2) << 23) * a.scale_log2;  // 2^(20 - k)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[g][t][k]));
                const float x = f.x * up, y = f.y * up;
                sum += x + y;
                qf[g][t][k] = k & 1 ? pack_half2(x, y) : pack_half2(16.f * x, 16.f * y);
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            sum *= 0x1p-20f;
            const float s0 = __shfl_sync(0xffffffffu, sum, 8 * j), s1 = __shfl_sync(0xffffffffu, sum, 8 * j + 4);
            qs[g][t] = pack_f32x2(s0, s1);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            unit[t][h] = __shfl_sync(0xffffffffu, down, 8 * j + 4 * h);
            const int qr = a.by_ratio.div(row0 + 8 * t + 2 * j + h);
            // (rows that are not there compute on zero queries and are never stored)
            limit[t][h] = qr >= nq ? (a.mask_kind == ET_MASK_ADDITIVE ? 0 : INT32_MAX)
                                   : (a.mask_kind == ET_MASK_CAUSAL ? len - nq + qr + 1 : len);
        }
    }

    float acc[NG][2][NT][4];  // [group][u]: features f = 2 u (elements 0, 1) and, times 16, 2 u + 1 (2, 3)
    uint64_t pm[NG][NT];      // sums of p (m + 8 s), two rows
    float l[NT][2], top[NT][2];  // sum of p, and the reference: -inf until the row sees a key
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            pm[g][t] = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[g][k >> 2][t][k & 3] = 0.f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) l[t][h] = 0.f, top[t][h] = -INFINITY;
    }

    const uint64_t minus_one = pack_f32x2(-1.f, -1.f);
    int tok0 = turn * TILE;
    for (int n = 0; n < mine; ++n, tok0 += turns * TILE) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        issue(n + STAGES - 1);  // into the slot that the previous tile left
        const uint8_t* st = ring + (n % STAGES) * S::STAGE;

        // ---- the lane's token: K's (s, m) to fp32; V's largest s, and whether all of V's are finite
        uint32_t vp[NG], odd_bits = 0, s_top = 0;
        {
            uint32_t kp[NG];
            lds_words<NG>(st + 2 * S::CODES + lane * 4 * NG, kp);
            lds_words<NG>(st + 2 * S::CODES + S::PARAMS + lane * 4 * NG, vp);
            if (tok0 + lane >= end) {  // hidden from every row: counts as zeros
#pragma unroll
                for (int g = 0; g < NG; ++g) kp[g] = vp[g] = 0u;
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&kp[g]));
                wide[lane * S::WIDE_LD + g] = make_float4(x.x, x.x, x.y, x.y);
                odd_bits |= (vp[g] & 0x7c007c00u) + 0x04000400u;  // (an exponent of all ones carries)
                s_top = max(s_top, vp[g] & 0x7fffu);
            }
        }
        const bool odd = __any_sync(0xffffffffu, (odd_bits & 0x80008000u) != 0);
        if (odd) {
            s_top = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (!q4::finite16(vp[g]) || !q4::finite16(vp[g] >> 16)) vp[g] = 0u;
                s_top = max(s_top, vp[g] & 0x7fffu);
            }
        }
        // every s of the token is < 2^e; e of tokens tau, tau + 8, ...
        const float e_mine = static_cast<float>(static_cast<int>(s_top >> 10) - 14);
        float e[2 * HALVES];
#pragma unroll
        for (int k = 0; k < 2 * HALVES; ++k) e[k] = __shfl_sync(0xffffffffu, e_mine, 8 * k + tau);
        __syncwarp();

        // ---- scores, in the row's units: [16-token block][token tau, tau + 8][row 2 j, 2 j + 1]
        float x[HALVES][NT][2][2];
#pragma unroll
        for (int bk = 0; bk < HALVES; ++bk) {
            uint32_t k0[NG], k1[NG];
            lds_words<NG>(st + (16 * bk + tau) * (16 * NG) + j * (4 * NG), k0);
            lds_words<NG>(st + (16 * bk + tau + 8) * (16 * NG) + j * (4 * NG), k1);
            uint64_t sum[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t) sum[t][0] = sum[t][1] = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t k0h = k0[g] >> 8, k1h = k1[g] >> 8;
                const uint32_t a0[4] = {k0[g] & q4::NIBBLES, k0[g] & (q4::NIBBLES << 4), k0h & q4::NIBBLES,
                                        k0h & (q4::NIBBLES << 4)};
                const uint32_t a1[4] = {k1[g] & q4::NIBBLES, k1[g] & (q4::NIBBLES << 4), k1h & q4::NIBBLES,
                                        k1h & (q4::NIBBLES << 4)};
                const float4 m0 = wide[(16 * bk + tau) * S::WIDE_LD + g];
                const float4 m1 = wide[(16 * bk + tau + 8) * S::WIDE_LD + g];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float d[4];
                    q4::mma0(d, a0[0], a1[0], a0[1], a1[1], qf[g][t][0], qf[g][t][1]);
                    q4::mma(d, a0[2], a1[2], a0[3], a1[3], qf[g][t][2], qf[g][t][3]);
                    sum[t][0] = fma_f32x2(pack_f32x2(d[0], d[1]), pack_f32x2(m0.x, m0.y),
                                          fma_f32x2(qs[g][t], pack_f32x2(m0.z, m0.w), sum[t][0]));
                    sum[t][1] = fma_f32x2(pack_f32x2(d[2], d[3]), pack_f32x2(m1.x, m1.y),
                                          fma_f32x2(qs[g][t], pack_f32x2(m1.z, m1.w), sum[t][1]));
                }
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                unpack_f32x2(sum[t][0], x[bk][t][0][0], x[bk][t][0][1]);
                unpack_f32x2(sum[t][1], x[bk][t][1][0], x[bk][t][1][1]);
            }
        }
        if (tok0 + TILE > least || a.mask_kind == ET_MASK_ADDITIVE) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float per_unit = LOG2E / unit[t][h];
                    const __half* mrow =
                        a.mask + static_cast<int64_t>(a.by_ratio.div(row0 + 8 * t + 2 * j + h)) * a.ldm;
#pragma unroll
                    for (int k = 0; k < 2 * HALVES; ++k) {
                        const int tok = tok0 + 8 * k + tau;
                        float& v = x[k >> 1][t][k & 1][h];
                        if (tok >= limit[t][h]) v = -INFINITY;
                        else if (a.mask_kind == ET_MASK_ADDITIVE) {
                            const float m = __half2float(__ldcg(mrow + tok));
                            v = m == -INFINITY ? -INFINITY : fmaf(m, per_unit, v);  // (-inf hides any score)
                        }
                    }
                }
        }

        uint32_t seen = 0;  // which of the scores are no -inf (an exponential of 0 may be a seen token's)
        if (odd) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 4 * HALVES; ++k)
                    if (x[k >> 2][t][(k >> 1) & 1][k & 1] != -INFINITY) seen |= 1u << (t * 4 * HALVES + k);
        }

        // ---- online softmax.  The reference moves only when a score plus e passes it by 6: the lanes then need not agree
        // on the tile's maximum, and p s < 2^6 is as good to fp16.
        float mx[NT][2];
        bool move = false;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[t][h] = fmaf(x[0][t][0][h], unit[t][h], e[0]);
#pragma unroll
                for (int k = 1; k < 2 * HALVES; ++k)
                    mx[t][h] = fmaxf(mx[t][h], fmaf(x[k >> 1][t][k & 1][h], unit[t][h], e[k]));
                move = move || mx[t][h] > top[t][h] + 6.f;
            }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                float shrink[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float m = fmaxf(mx[t][h], __shfl_xor_sync(0xffffffffu, mx[t][h], 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    m = fmaxf(m, top[t][h]);
                    // (a row that has seen nothing keeps sums of zero)
                    shrink[h] = top[t][h] == -INFINITY ? 1.f : exp2f(top[t][h] - m);
                    top[t][h] = m;
                    l[t][h] *= shrink[h];
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    pm[g][t] = mul_f32x2(pm[g][t], pack_f32x2(shrink[0], shrink[1]));
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[g][k >> 2][t][k & 3] *= shrink[k & 1];
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float ref = top[t][h] == -INFINITY ? 0.f : top[t][h];
#pragma unroll
                for (int k = 0; k < 2 * HALVES; ++k) {
                    float& v = x[k >> 1][t][k & 1][h];
                    v = exp2_approx(fmaf(v, unit[t][h], -ref));
                    l[t][h] += v;
                }
            }
        uint64_t px[HALVES][NT][2];  // the same, rows in pairs
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 2 * HALVES; ++k)
                px[k >> 1][t][k & 1] = pack_f32x2(x[k >> 1][t][k & 1][0], x[k >> 1][t][k & 1][1]);
        if (odd) {  // a group of V that is not finite: NaN for the rows that see it, however little, and for no other
            const uint32_t* raw = reinterpret_cast<const uint32_t*>(st + 2 * S::CODES + S::PARAMS);
#pragma unroll
            for (int k = 0; k < 2 * HALVES; ++k) {
                const int tok = 8 * k + tau;
                if (tok0 + tok >= end) continue;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t w = raw[tok * NG + g];
                    if (q4::finite16(w) && q4::finite16(w >> 16)) continue;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float p0, p1;
                        unpack_f32x2(pm[g][t], p0, p1);
                        if (seen >> (t * 4 * HALVES + 2 * k) & 1) p0 = NAN;
                        if (seen >> (t * 4 * HALVES + 2 * k + 1) & 1) p1 = NAN;
                        pm[g][t] = pack_f32x2(p0, p1);
                    }
                }
            }
        }

        // ---- V's (s, m + 8 s) to fp32, in K's place
        __syncwarp();
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&vp[g]));
            const float m = fmaf(8.f, v.x, v.y);
            wide[lane * S::WIDE_LD + g] = make_float4(v.x, v.x, m, m);
        }
        __syncwarp();

        // ---- second product
#pragma unroll
        for (int bk = 0; bk < HALVES; ++bk) {
            uint32_t vu[4][(NG + 1) / 2];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                lds_units<NG>(st + S::CODES + (16 * bk + j + 4 * u) * (16 * NG) + i * (2 * NG), vu[u]);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t sel = g & 1 ? 0x7632u : 0x5410u;
                const uint32_t w0 = __byte_perm(vu[0][g / 2], vu[1][g / 2], sel);
                const uint32_t w1 = __byte_perm(vu[2][g / 2], vu[3][g / 2], sel);
                const uint32_t w0h = w0 >> 8, w1h = w1 >> 8;
                const uint32_t f0 = q4::centred(w0), f1 = q4::centred16(w0), f2 = q4::centred(w0h),
                               f3 = q4::centred16(w0h);
                const uint32_t g0 = q4::centred(w1), g1 = q4::centred16(w1), g2 = q4::centred(w1h),
                               g3 = q4::centred16(w1h);
                const float4 m0 = wide[(16 * bk + tau) * S::WIDE_LD + g];
                const float4 m1 = wide[(16 * bk + tau + 8) * S::WIDE_LD + g];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    uint32_t hi[2], lo[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float4& m = h ? m1 : m0;
                        const uint64_t p = px[bk][t][h];
                        const uint64_t ps = mul_f32x2(p, pack_f32x2(m.x, m.y));
                        pm[g][t] = fma_f32x2(p, pack_f32x2(m.z, m.w), pm[g][t]);
                        float p0, p1;
                        unpack_f32x2(ps, p0, p1);
                        const uint32_t top16 = pack_half2(p0, p1);
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&top16));
                        unpack_f32x2(fma_f32x2(pack_f32x2(back.x, back.y), minus_one, ps), p0, p1);
                        hi[h] = transposed(top16);
                        lo[h] = transposed(pack_half2(p0, p1));
                    }
                    q4::mma(acc[g][0][t], f0, f1, g0, g1, hi[0], hi[1]);
                    q4::mma(acc[g][1][t], f2, f3, g2, g3, hi[0], hi[1]);
                    q4::mma(acc[g][0][t], f0, f1, g0, g1, lo[0], lo[1]);
                    q4::mma(acc[g][1][t], f2, f3, g2, g3, lo[0], lo[1]);
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with its ring: it becomes the exchange area

    // ---- join the warps: [warp][row][D] sums and [warp][row][2] (reference, sum of p)
    float* xs = reinterpret_cast<float*>(smem);
    constexpr int ROWS = 8 * NT;
    float* xml = xs + WARPS * ROWS * D;
    auto over_tokens = [](float v) {
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        return v + __shfl_xor_sync(0xffffffffu, v, 16);
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int row = warp * ROWS + 8 * t + 2 * j;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[t][h] = over_tokens(l[t][h]);
            if (i == 0) {
                // (a row whose every score is NaN has no maximum, but is not empty)
                xml[2 * (row + h)] = l[t][h] != l[t][h] && top[t][h] == -INFINITY ? 0.f : top[t][h];
                xml[2 * (row + h) + 1] = l[t][h];
            }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float m[2];
            unpack_f32x2(pm[g][t], m[0], m[1]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                m[h] = over_tokens(m[h]);
                *reinterpret_cast<float4*>(xs + (row + h) * D + 32 * g + 4 * i) =
                    make_float4(acc[g][0][t][h] + m[h], fmaf(acc[g][0][t][2 + h], 0.0625f, m[h]),
                                acc[g][1][t][h] + m[h], fmaf(acc[g][1][t][2 + h], 0.0625f, m[h]));
            }
        }
    }
    __syncthreads();
    // eight features of a row per thread and step: the warps', then (few splits) the blocks' of a cluster
    float* mine_x = xml + 2 * WARPS * ROWS;  // this block's sums [row][D] and (reference, sum of p)
    float* mine_ml = mine_x + ROWS * D;
    static_assert((WARPS + 1) * ROWS * (D + 2) * 4 <= S::TOTAL, "exchange area");
    const bool clustered = a.splits > 1 && a.splits <= MAX_CLUSTER;
    for (int u = threadIdx.x; u < ROWS * (D / 8); u += THREADS) {
        const int r = u / (D / 8), d = (u - r * (D / 8)) * 8;
        const int rr = row0 + r, qi = a.by_ratio.div(rr), head = kvh * a.ratio + rr - qi * a.ratio;
        if (qi >= nq) continue;
        float o[8], top_all, sum;
        join_partials<WARPS>(WARPS, o, top_all, sum, [&](int w) { return xml + 2 * (w * ROWS + r); },
                             [&](int w) { return xs + (w * ROWS + r) * D + d; });
        const int64_t row = static_cast<int64_t>(b) * a.seq + qi;
        if (clustered) {
            store8(mine_x + r * D + d, o);
            if (d == 0) {
                mine_ml[2 * r] = top_all;
                mine_ml[2 * r + 1] = sum;
            }
        } else if (a.splits > 1) {
            const int64_t at = (static_cast<int64_t>(split) * a.batch * a.seq + row) * a.nhead + head;
            store8(a.part + at * D + d, o);
            if (d == 0) {
                a.part_ml[2 * at] = top_all;
                a.part_ml[2 * at + 1] = sum;
            }
        } else if (d < a.c.dh[1]) {
            store_z(a.Z + row * a.ldz + head * a.c.dh[1] + d, o, top_all, sum);
        }
    }
    if (!clustered) return;
    __syncwarp();
    cluster_sync_all();
    const uint32_t x32 = smem_u32(mine_x), ml32 = smem_u32(mine_ml);
    static_assert(ROWS * (D / 8) <= 2 * THREADS, "one step of the cluster's threads");
    const int u = threadIdx.x * a.splits + split;
    const int r = u / (D / 8), d = (u - r * (D / 8)) * 8;
    const int rr = row0 + r, qi = a.by_ratio.div(rr), head = kvh * a.ratio + rr - qi * a.ratio;
    const bool there = r < ROWS && qi < nq && d < a.c.dh[1];
    float o[8], top_all, sum;
    if (there)
        join_partials<MAX_CLUSTER>(a.splits, o, top_all, sum,
                                   [&](int c) { return map_to_cta(ml32 + 8 * r, c); },
                                   [&](int c) { return map_to_cta(x32 + (r * D + d) * 4, c); });
    // No block leaves while another reads its shared memory.  (Arriving before the result is stored, so that the barrier
    // does not wait for the store: 1 x 1024 tokens, 32/8 heads of 128 6.5 us for 6.6.)
    __syncwarp();
    cluster_arrive();
    if (there) store_z(a.Z + (static_cast<int64_t>(b) * a.seq + qi) * a.ldz + head * a.c.dh[1] + d, o, top_all, sum);
    __syncwarp();
    cluster_wait();
}

// Joins the splits' partial results: a warp per (row, head), four features per lane.  What it takes is one trip to
// memory and the launch; the sums are asked for before their factors are known.
__global__ void __launch_bounds__(64) attention_kv4_join_kernel(const AttArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int all = a.batch * a.seq * a.nhead, at = blockIdx.x * 2 + (threadIdx.x >> 5);
    if (at >= all) return;
    const int row = at / a.nhead, head = at - row * a.nhead, b = row / a.seq;
    if (a.q_len && row - b * a.seq >= __ldcg(a.q_len + b)) return;
    const int lane = threadIdx.x & 31, D = 32 * a.c.ng;
    const float4* part = reinterpret_cast<const float4*>(a.part + static_cast<int64_t>(at) * D) + (4 * lane < D ? lane : 0);
    const int64_t next = static_cast<int64_t>(all) * D / 4;  // from a split to the next
    auto load = [&](float4(&v)[JOIN_AHEAD], int s0) {
#pragma unroll
        for (int k = 0; k < JOIN_AHEAD; ++k)  // (past the last split that one again: its factor is 0 below)
            v[k] = __ldcg(part + (s0 + k < a.splits ? s0 + k : a.splits - 1) * next);
    };
    float4 v[JOIN_AHEAD];
    load(v, 0);
    // splits <= 64: two of (reference, sum of p) per lane
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at;
    float2 m0 = make_float2(-INFINITY, 0.f), m1 = m0;
    if (lane < a.splits) m0 = __ldcg(ml + static_cast<int64_t>(lane) * all);
    if (lane + 32 < a.splits) m1 = __ldcg(ml + static_cast<int64_t>(lane + 32) * all);
    float top = fmaxf(m0.x, m1.x);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float f0 = m0.x == -INFINITY ? 0.f : exp2f(m0.x - top), f1 = m1.x == -INFINITY ? 0.f : exp2f(m1.x - top);
    float sum = m0.y * f0 + m1.y * f1;
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0;;) {
#pragma unroll
        for (int k = 0; k < JOIN_AHEAD; ++k) {
            const int s = s0 + k;
            const float f = __shfl_sync(0xffffffffu, s < 32 ? f0 : f1, s & 31);
            if (s < a.splits) {  // (a split that saw nothing has sums of 0; one far below the others may hold a NaN)
                o.x = fmaf(v[k].x, f, o.x);
                o.y = fmaf(v[k].y, f, o.y);
                o.z = fmaf(v[k].z, f, o.z);
                o.w = fmaf(v[k].w, f, o.w);
            }
        }
        if ((s0 += JOIN_AHEAD) >= a.splits) break;
        load(v, s0);
    }
    if (4 * lane < a.c.dh[1]) {
        const float inv = top == -INFINITY ? 0.f : 1.f / sum;
        uint2 z;
        z.x = pack_half2(o.x * inv, o.y * inv);
        z.y = pack_half2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(a.Z + static_cast<int64_t>(row) * a.ldz + head * a.c.dh[1] + 4 * lane) = z;
    }
}

// Thread blocks along the sequence: as many as are resident at once (a second wave would run next to nothing: 4 x 8
// heads x 32768 tokens took 91 us in 416 blocks on 296 places), of MIN_CHUNK tokens at least (7 sequences of 777
// tokens: 8.4 us with 256, 9.5 with 512, 12.1 with 1024).
int pick_splits(int64_t blocks, int max_len, int ng, int nt) {
    const int sms = sm_count() > 0 ? sm_count() : 148;
    int64_t s = blocks_per_sm(ng, nt) * sms / blocks;
    const int64_t most = (max_len + MIN_CHUNK - 1) / MIN_CHUNK;
    s = s < most ? s : most;
    return static_cast<int>(s < 1 ? 1 : (s > MAX_SPLITS ? MAX_SPLITS : s));
}

struct AttPlan {
    int nt, tiles, splits;
    size_t part, ml;
};
AttPlan plan_att(const Kv4View& v, int batch, int seq, int nhead, int max_len) {
    AttPlan p;
    const int64_t rows = static_cast<int64_t>(seq) * (nhead / v.nkv);
    p.nt = rows > 8 ? 2 : 1;
    p.tiles = static_cast<int>((rows + 8 * p.nt - 1) / (8 * p.nt));
    p.splits = pick_splits(static_cast<int64_t>(p.tiles) * v.nkv * batch, max_len, v.ng, p.nt);
    const size_t all = static_cast<size_t>(batch) * seq * nhead;
    p.part = p.splits > MAX_CLUSTER ? p.splits * all * 32 * v.ng * sizeof(float) : 0;
    p.ml = p.splits > MAX_CLUSTER ? p.splits * all * 2 * sizeof(float) : 0;
    return p;
}

template <int NG, int NT>
int launch_att(const AttArgs& a, cudaStream_t stream) {
    auto kern = attention_kv4_kernel<NG, NT>;
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<NG, NT>::TOTAL) != cudaSuccess)
            return ET_ERR_CUDA;
        attr_set[dev] = true;
    }
    const dim3 grid(a.splits, a.tiles * a.c.nkv, a.batch);
    // Clusters of up to 4 / of up to 8 / the second kernel always, in us: 1 x 512 tokens, 12 heads 4.6 / 4.8 / 5.5;
    // 8 x 1024 8.2 / 8.8 / 9.3; 16 x 2000 18.1 / 18.4 / 19.1; 2 x 64 queries over 1025 tokens 13.6 / 12.8 / 13.7.  (Of
    // 13 blocks they found no places: 4 x 32768 tokens 78 for 56.)
    if (a.splits == 1 || a.splits > MAX_CLUSTER)
        return launch_kernel(kern, grid, dim3(THREADS), Shape<NG, NT>::TOTAL, stream, a) == cudaSuccess ? ET_OK : ET_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Shape<NG, NT>::TOTAL;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(a.splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    count_launch();
    return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? ET_OK : ET_ERR_CUDA;
}

}  // namespace
}  // namespace et

extern "C" {

size_t et_attention_kv4_workspace_bytes(const et_kv4_t* cache, int batch, int seq, int nhead, int max_len) {
    et::Kv4View v;
    if (et::kv4_view(cache, v, false) != ET_OK || et::kv4_check_attention(v, batch, seq, nhead, max_len) != ET_OK) return 0;
    const et::AttPlan p = et::plan_att(v, batch, seq, nhead, max_len);
    return p.part + p.ml;
}

int et_attention_kv4_fwd(const et_kv4_t* cache, const et_half* Q, et_half* Z, const int32_t* table, int table_ld,
                         const int32_t* kv_len, const int32_t* q_len, int batch, int seq, int nhead, int ldq,
                         int ldz, int max_len, int mask_kind, const et_half* mask, int ldm, float scale,
                         void* workspace, size_t workspace_bytes, et_stream stream) {
    et::AttArgs a = {};
    int st = et::kv4_view(cache, a.c, true);
    if (st != ET_OK) return st;
    if (!Q || !Z || !table || !kv_len || table_ld <= 0) return ET_ERR_INVALID_ARG;
    if ((st = et::kv4_check_attention(a.c, batch, seq, nhead, max_len)) != ET_OK) return st;
    if (mask_kind != ET_MASK_NONE && mask_kind != ET_MASK_CAUSAL && mask_kind != ET_MASK_ADDITIVE)
        return ET_ERR_INVALID_ARG;
    if (mask_kind == ET_MASK_ADDITIVE && (!mask || ldm < max_len)) return ET_ERR_INVALID_ARG;
    if (!(scale >= 0x1p-64f && scale <= 0x1p64f)) return ET_ERR_INVALID_ARG;  // (masks are divided by it)
    if (static_cast<int64_t>(table_ld) << a.c.page_shift < max_len) return ET_ERR_SHAPE;
    if (ldq % 8 || ldz % 8 || ldq < static_cast<int64_t>(nhead) * a.c.dh[0] || ldz < static_cast<int64_t>(nhead) * a.c.dh[1])
        return ET_ERR_SHAPE;
    if (!et::aligned16(Q) || !et::aligned16(Z)) return ET_ERR_ALIGNMENT;
    const et::AttPlan p = et::plan_att(a.c, batch, seq, nhead, max_len);
    if (p.splits > et::MAX_CLUSTER) {
        if (!workspace || workspace_bytes < p.part + p.ml) return ET_ERR_WORKSPACE;
        if (!et::aligned16(workspace)) return ET_ERR_ALIGNMENT;
    }
    a.Q = reinterpret_cast<const __half*>(Q);
    a.Z = reinterpret_cast<__half*>(Z);
    a.table = table;
    a.kv_len = kv_len;
    a.q_len = q_len;
    a.mask = reinterpret_cast<const __half*>(mask);
    a.part = static_cast<float*>(workspace);
    a.part_ml = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + p.part);
    a.table_ld = table_ld;
    a.batch = batch, a.seq = seq, a.nhead = nhead, a.ratio = nhead / a.c.nkv;
    a.ldq = ldq, a.ldz = ldz, a.ldm = ldm, a.max_len = max_len;
    a.mask_kind = mask_kind;
    a.by_ratio = et::FastDiv(static_cast<uint32_t>(a.ratio));
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.scale_log2 = scale * et::LOG2E;
    a.err_word = et::device_error_word();
    if (!a.err_word) return ET_ERR_NO_DEVICE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (a.c.ng * 2 + p.nt) {
        case 3: st = et::launch_att<1, 1>(a, s); break;
        case 4: st = et::launch_att<1, 2>(a, s); break;
        case 5: st = et::launch_att<2, 1>(a, s); break;
        case 6: st = et::launch_att<2, 2>(a, s); break;
        case 7: st = et::launch_att<3, 1>(a, s); break;
        case 8: st = et::launch_att<3, 2>(a, s); break;
        case 9: st = et::launch_att<4, 1>(a, s); break;
        default: st = et::launch_att<4, 2>(a, s); break;
    }
    if (st != ET_OK || p.splits <= et::MAX_CLUSTER) return st;
    const int64_t all = static_cast<int64_t>(batch) * seq * nhead;
    return et::launch_kernel(et::attention_kv4_join_kernel, dim3(static_cast<unsigned>((all + 1) / 2)), dim3(64), 0, s,
                             a) == cudaSuccess
               ? ET_OK
               : ET_ERR_CUDA;
}

}  // extern "C"
