// Attention of new queries over a key/value cache held in 4 bits (see quant4.cuh for the numbers, et_b200.h for
// the layout).
//
// Mathematics.  With k_t = c s + m per group g of 32 features, the score of row i is
//     q_i . k_t = sum_g ( s_g(t) (q_i . c_t)_g + m_g(t) (sum of q_i over g) ),
// so the tensor core multiplies fp16 queries by codes (exact; fp32 sums) and scale and minimum are applied to
// its results.  For the second product the scale goes to the probability instead,
//     out[d in g] = ( sum_t (p_t s_g(t)) (c_t[d] - 8)  +  sum_t p_t (m_g(t) + 8 s_g(t)) ) / sum_t p_t,
// with p s split into two fp16 numbers (22 bits) that share the fragment of one product: rows 0-7 of the
// 16-row operand hold the high parts, rows 8-15 the low ones (up to eight query rows), or two products (16).
// (Codes less 8: sums of codes of one sign grow with the sequence while the output shrinks, and the tensor core
// cuts its fp32 sums: at 32768 tokens that cost half of the result's own rounding again, 3.2e-4 for 2.1e-4.)
// The softmax is online; its reference is the running maximum of the scaled scores plus the exponent of the
// running largest s, so that p s <= 1 whatever the magnitude of V.
//
// A thread block owns up to 16 query rows that share a key/value head (the heads of a group times the query tokens) and a
// chunk of the sequence; its four warps take 32-token tiles in turn, each with a ring of asynchronous copies of its
// own (page contents land in shared memory as they are; no thread waits for another warp in the loop).  With
// few rows the sequence is split over blocks whose partial results a second kernel joins.
//
// Layout of a tile in registers (lane = 4 i + j): the cache stores rows so that a lane's words are consecutive.  K:
// lane (i, j) holds word j of every group of token tau(i) = (i >> 1) + 4 (i & 1), which makes its score columns
// 2 j, 2 j + 1 tokens j and j + 4; V: unit i of every group of tokens j, j + 4, j + 8, j + 12 - the order in which those scores
// sit in the second product's operand.
#include "kernels.h"
#include "kv4.h"
#include "quant4.cuh"

namespace et {
namespace {

constexpr int TILE = 32;      // tokens of a warp's tile
constexpr int WARPS = 4;
constexpr int STAGES = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int MAX_SPLITS = 64;
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
    int rows, tiles;  // query rows per (sequence, key/value head), row tiles
    int splits;
    float scale_log2;
    int* err_word;
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;  // 0: zeros are written, nothing is read
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(n) : "memory");
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

template <int NG>
struct Smem {
    static constexpr int CODES = TILE * 16 * NG, PARAMS = TILE * 4 * NG;
    static constexpr int STAGE = 2 * (CODES + PARAMS);  // K codes, V codes, K params, V params
    static constexpr int RING = STAGES * STAGE;
    static constexpr int WIDE = TILE * NG * 16;  // (s, m) of K and of V as fp32
    static constexpr int WARP = RING + WIDE;
    static constexpr int TOTAL = WARPS * WARP;
};

// RT: 8-row tiles (1: the 16-row operand's other half carries the low parts; 2: 16 query rows).
template <int NG, int RT>
__global__ void __launch_bounds__(THREADS, NG <= 2 ? 4 : (NG == 3 ? 3 : 2)) attention_kv4_kernel(const AttArgs a) {
    using S = Smem<NG>;
    constexpr int D = 32 * NG;
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = lane >> 2, j = lane & 3;
    uint8_t* ring = smem + warp * S::WARP;
    float4* wide = reinterpret_cast<float4*>(ring + S::RING);  // [token][group] sK, mK, sV, mV + 8 sV

    pdl_wait();
    pdl_launch_dependents();

    const int split = blockIdx.x;
    const int rt = blockIdx.y % a.tiles, kvh = blockIdx.y / a.tiles;
    const int b = blockIdx.z;
    int len = __ldcg(a.kv_len + b);
    if (len > a.max_len) {
        if (threadIdx.x == 0) atomicCAS(a.err_word, 0, DEV_BAD_PAGE);
        len = a.max_len;
    }
    len = len < 0 ? 0 : len;
    int nq = a.q_len ? __ldcg(a.q_len + b) : a.seq;
    nq = nq < 0 ? 0 : (nq > a.seq ? a.seq : nq);

    // ---- rows: row r of the tile is query token r / ratio, head kvh * ratio + r % ratio
    const int row0 = rt * 8 * RT;
    if (row0 >= nq * a.ratio) return;  // (rows are ordered by query token)
    int limit[RT];                     // tokens that a row sees
    uint32_t qf[NG][RT][4];            // its queries: features 32 g + 8 j .. + 8
    float qs[NG][RT];                  // sum of the group's queries times 2^-24 (the codes carry that factor)
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int r = row0 + 8 * t + i;
        const int qi = r / a.ratio, head = kvh * a.ratio + r % a.ratio;
        const bool live = qi < nq;
        // (rows that are not there compute on zero queries and are never stored)
        limit[t] = !live ? (a.mask_kind == ET_MASK_ADDITIVE ? 0 : INT32_MAX)
                         : (a.mask_kind == ET_MASK_CAUSAL ? len - nq + qi + 1 : len);
        const __half* q = a.Q + (static_cast<int64_t>(b) * a.seq + qi) * a.ldq + head * a.c.dh[0] + 8 * j;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live && 32 * g + 8 * j < a.c.dh[0]) v = __ldcg(reinterpret_cast<const uint4*>(q + 32 * g));
            qf[g][t][0] = v.x, qf[g][t][1] = v.y, qf[g][t][2] = v.z, qf[g][t][3] = v.w;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[g][t][k]));
                sum += f.x + f.y;
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qs[g][t] = sum * 0x1p-24f;
        }
    }
    int most, least;  // the largest and smallest limit: those of the last and first row
    {
        const int last = (row0 + 8 * RT < nq * a.ratio ? row0 + 8 * RT : nq * a.ratio) - 1;
        if (a.mask_kind == ET_MASK_CAUSAL) {
            least = len - nq + row0 / a.ratio + 1;
            most = len - nq + last / a.ratio + 1;
        } else {
            least = most = len;
        }
        most = most < 0 ? 0 : most;
    }
    // this block's chunk of the sequence, and the warp's tiles in it
    const int per = ((most + a.splits - 1) / a.splits + TILE - 1) / TILE * TILE;
    const int64_t first64 = static_cast<int64_t>(split) * per;
    const int first = first64 < most ? static_cast<int>(first64) : most;
    const int end = first + per < most ? first + per : most;
    const int ntile = (end - first + TILE - 1) / TILE;
    const int mine = ntile > warp ? (ntile - warp + WARPS - 1) / WARPS : 0;  // tiles warp, warp + 4, ...

    // ---- page numbers of 16 tiles at a time, one half tile (16 tokens) to a lane
    const int* table = a.table + static_cast<int64_t>(b) * a.table_ld;
    auto page_of = [&](int n) {  // of half tile `lane` of the 16 tiles from tile n on; -1: nothing to read
        const int pos = first + ((n + (lane >> 1)) * WARPS + warp) * TILE + (lane & 1) * 16;
        if (pos >= end || n + (lane >> 1) >= mine) return -1;
        const int id = kv4_page(a.c, table, a.table_ld, pos);
        if (id < 0) atomicCAS(a.err_word, 0, DEV_BAD_PAGE);
        return id;
    };
    int pages = page_of(0), pages_next = page_of(16);
    // copies tile n of this warp (call with n = 0, 1, 2, ... in order)
    auto issue = [&](int n) {
        if (n < mine) {
            if (n != 0 && (n & 15) == 0) {
                pages = pages_next;
                pages_next = page_of(n + 16);
            }
            uint8_t* st = ring + (n % STAGES) * S::STAGE;
            const int pos = first + (n * WARPS + warp) * TILE;
            const int id0 = __shfl_sync(0xffffffffu, pages, (n & 15) * 2);
            const int id1 = __shfl_sync(0xffffffffu, pages, (n & 15) * 2 + 1);
            // rows of the two half tiles (of 0 where nothing is read: any address inside the arrays will do)
            const int64_t r0 = id0 < 0 ? 0 : kv4_row(a.c, id0, pos, kvh);
            const int64_t r1 = id1 < 0 ? 0 : kv4_row(a.c, id1, pos + 16, kvh);
#pragma unroll
            for (int of = 0; of < 2; ++of) {
#pragma unroll
                for (int u = 0; u < NG; ++u) {  // 32 NG pieces of codes, half of them per half tile
                    const int p = u * 32 + lane;
                    const bool hi = p >= 16 * NG;
                    const int id = hi ? id1 : id0;
                    const uint8_t* src = a.c.codes[of] + (hi ? r1 : r0) * (16 * NG) + (hi ? p - 16 * NG : p) * 16;
                    cp_async16(st + of * S::CODES + p * 16, id < 0 ? a.c.codes[of] : src, id >= 0);
                }
                // 8 NG pieces of parameters
                if (lane < 8 * NG) {
                    const bool hi = lane >= 4 * NG;
                    const int id = hi ? id1 : id0;
                    const uint8_t* base = reinterpret_cast<const uint8_t*>(a.c.params[of]);
                    const uint8_t* src = base + (hi ? r1 : r0) * (4 * NG) + (hi ? lane - 4 * NG : lane) * 16;
                    cp_async16(st + 2 * S::CODES + of * S::PARAMS + lane * 16, id < 0 ? base : src, id >= 0);
                }
            }
        }
        cp_async_commit();  // (an empty group past the last tile, so that the count stays)
    };

    float acc[NG][4][4];  // [group][f]: the second product's fragments
    float pm[NG][RT], l[RT], top[RT];
    float e = -24.f;  // exponent: every s so far is <= 2^e
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int f = 0; f < 4; ++f)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[g][f][k] = 0.f;
#pragma unroll
        for (int t = 0; t < RT; ++t) pm[g][t] = 0.f;
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) l[t] = 0.f, top[t] = -INFINITY;

#pragma unroll
    for (int n = 0; n < STAGES - 1; ++n) issue(n);

    for (int n = 0; n < mine; ++n) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        issue(n + STAGES - 1);  // into the slot that the previous tile left
        const uint8_t* st = ring + (n % STAGES) * S::STAGE;
        const int tok0 = first + (n * WARPS + warp) * TILE;

        // ---- (s, m) of token `lane` to fp32; tokens past the end count as zeros
        bool odd = false;
        uint32_t s_top = 0;
        {
            uint32_t kp[NG], vp[NG];
            lds_words<NG>(st + 2 * S::CODES + lane * 4 * NG, kp);
            lds_words<NG>(st + 2 * S::CODES + S::PARAMS + lane * 4 * NG, vp);
            const bool in = tok0 + lane < end;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float2 k = __half22float2(*reinterpret_cast<const __half2*>(&kp[g]));
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&vp[g]));
                const bool fine = q4::finite16(vp[g]) && q4::finite16(vp[g] >> 16);
                odd = odd || (in && !fine);
                const uint32_t bits = in && fine ? __float_as_uint(fabsf(v.x)) : 0u;
                s_top = bits > s_top ? bits : s_top;
                wide[lane * NG + g] =
                    in ? make_float4(k.x, k.y, v.x, fmaf(8.f, v.x, v.y)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
        odd = __any_sync(0xffffffffu, odd);
        s_top = __reduce_max_sync(0xffffffffu, s_top);
        // 2^(exponent + 1) >= s
        const float e_new = fmaxf(e, static_cast<float>(static_cast<int>(s_top >> 23) - 126));
        __syncwarp();

        // ---- scores
        float x[2][RT][4];  // [16-token block][row][token j, j + 4, j + 8, j + 12 of the block]
#pragma unroll
        for (int bk = 0; bk < 2; ++bk)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                const int base = 16 * bk + 8 * nt;
                uint32_t kw[NG];
                lds_words<NG>(st + (base + (i >> 1) + 4 * (i & 1)) * (16 * NG) + j * (4 * NG), kw);
                float s0[RT], s1[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) s0[t] = s1[t] = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    float d[4];
                    q4::mma0(d, qf[g][0][0], RT > 1 ? qf[g][RT - 1][0] : 0u, qf[g][0][1],
                             RT > 1 ? qf[g][RT - 1][1] : 0u, kw[g] & q4::NIBBLES, (kw[g] >> 4) & q4::NIBBLES);
                    q4::mma(d, qf[g][0][2], RT > 1 ? qf[g][RT - 1][2] : 0u, qf[g][0][3],
                            RT > 1 ? qf[g][RT - 1][3] : 0u, (kw[g] >> 8) & q4::NIBBLES, (kw[g] >> 12) & q4::NIBBLES);
                    const float2 p0 = *reinterpret_cast<const float2*>(&wide[(base + j) * NG + g]);
                    const float2 p1 = *reinterpret_cast<const float2*>(&wide[(base + j + 4) * NG + g]);
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        s0[t] = fmaf(d[2 * t], p0.x, fmaf(qs[g][t], p0.y, s0[t]));
                        s1[t] = fmaf(d[2 * t + 1], p1.x, fmaf(qs[g][t], p1.y, s1[t]));
                    }
                }
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    x[bk][t][2 * nt] = s0[t] * a.scale_log2;
                    x[bk][t][2 * nt + 1] = s1[t] * a.scale_log2;
                }
            }
        if (tok0 + TILE > least || a.mask_kind == ET_MASK_ADDITIVE) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int r = row0 + 8 * t + i;
                const __half* mrow = a.mask + static_cast<int64_t>(r / a.ratio) * a.ldm;
#pragma unroll
                for (int bk = 0; bk < 2; ++bk)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int tok = tok0 + 16 * bk + j + 4 * u;
                        if (tok >= limit[t]) x[bk][t][u] = -INFINITY;
                        else if (a.mask_kind == ET_MASK_ADDITIVE) {
                            const float m = __half2float(__ldcg(mrow + tok));
                            // (-inf hides the key whatever its score)
                            x[bk][t][u] = m == -INFINITY ? -INFINITY : fmaf(m, LOG2E, x[bk][t][u]);
                        }
                    }
            }
        }

        // ---- online softmax
        float ref[RT];
        bool moved = false;
        float scale_old[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            float mx = -INFINITY;
#pragma unroll
            for (int bk = 0; bk < 2; ++bk)
#pragma unroll
                for (int u = 0; u < 4; ++u) mx = fmaxf(mx, x[bk][t][u]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            mx = fmaxf(mx, top[t]);
            // a row that has seen nothing yet keeps sums of zero, whatever its reference
            const float now = mx == -INFINITY ? 0.f : mx;
            scale_old[t] = top[t] == -INFINITY ? 1.f : exp2f(top[t] - now + e - e_new);
            moved = moved || scale_old[t] != 1.f;
            top[t] = mx;
            ref[t] = now + e_new;
        }
        e = e_new;
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                l[t] *= scale_old[t];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    pm[g][t] *= scale_old[t];
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        acc[g][f][2 * t] *= scale_old[t];
                        acc[g][f][2 * t + 1] *= scale_old[t];
                        if (RT == 1) {
                            acc[g][f][2] *= scale_old[t];
                            acc[g][f][3] *= scale_old[t];
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int bk = 0; bk < 2; ++bk)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    x[bk][t][u] = exp2_approx(x[bk][t][u] - ref[t]);
                    l[t] += x[bk][t][u];
                }

        // ---- second product
#pragma unroll
        for (int bk = 0; bk < 2; ++bk) {
            uint32_t vu[4][(NG + 1) / 2];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                lds_units<NG>(st + S::CODES + (16 * bk + j + 4 * u) * (16 * NG) + i * (2 * NG), vu[u]);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t hi[RT][2], lo[RT][2];
                float2 sm[4];
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    sm[u] = *(reinterpret_cast<const float2*>(&wide[(16 * bk + j + 4 * u) * NG + g]) + 1);
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    float ps[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const float p = x[bk][t][u];
                        ps[u] = p * sm[u].x;
                        float add = p * sm[u].y;
                        if (odd && p == 0.f) ps[u] = add = 0.f;  // a hidden key's NaN stays hidden
                        pm[g][t] += add;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        hi[t][h] = pack_half2(ps[2 * h], ps[2 * h + 1]);
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&hi[t][h]));
                        lo[t][h] = pack_half2(ps[2 * h] - back.x, ps[2 * h + 1] - back.y);
                    }
                }
                const uint32_t sel = g & 1 ? 0x7632u : 0x5410u;
                const uint32_t w0 = __byte_perm(vu[0][g / 2], vu[1][g / 2], sel);
                const uint32_t w1 = __byte_perm(vu[2][g / 2], vu[3][g / 2], sel);
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    const uint32_t b0 = q4::centred(w0 >> (4 * f)), b1 = q4::centred(w1 >> (4 * f));
                    if (RT == 1) {
                        q4::mma(acc[g][f], hi[0][0], lo[0][0], hi[0][1], lo[0][1], b0, b1);
                    } else {
                        q4::mma(acc[g][f], hi[0][0], hi[RT - 1][0], hi[0][1], hi[RT - 1][1], b0, b1);
                        q4::mma(acc[g][f], lo[0][0], lo[RT - 1][0], lo[0][1], lo[RT - 1][1], b0, b1);
                    }
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();  // every warp is done with its ring: it becomes the exchange area

    // ---- join the warps: [warp][row][D] sums and [warp][row][2] (reference, sum of p)
    float* xs = reinterpret_cast<float*>(smem);
    constexpr int ROWS = 8 * RT;
    static_assert(WARPS * ROWS * (D + 2) * 4 <= S::TOTAL, "exchange area");
    float* xml = xs + WARPS * ROWS * D;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        l[t] += __shfl_xor_sync(0xffffffffu, l[t], 1);
        l[t] += __shfl_xor_sync(0xffffffffu, l[t], 2);
        const int row = warp * ROWS + 8 * t + i;
        if (j == 0) {
            // (a row whose every score is NaN has no maximum, but is not empty)
            xml[2 * row] = l[t] != l[t] && top[t] == -INFINITY ? 0.f : top[t] + e;
            xml[2 * row + 1] = l[t];
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float m = pm[g][t];
            m += __shfl_xor_sync(0xffffffffu, m, 1);
            m += __shfl_xor_sync(0xffffffffu, m, 2);
            float o[2][4];
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float v = RT == 1 ? acc[g][f][h] + acc[g][f][2 + h] : acc[g][f][2 * t + h];
                    o[h][f] = v + m;
                }
            float4* p = reinterpret_cast<float4*>(xs + row * D + 32 * g + 8 * j);
            p[0] = make_float4(o[0][0], o[0][1], o[0][2], o[0][3]);
            p[1] = make_float4(o[1][0], o[1][1], o[1][2], o[1][3]);
        }
    }
    __syncthreads();
    // eight features of a row per thread and step
    for (int u = threadIdx.x; u < ROWS * (D / 8); u += THREADS) {
        const int r = u / (D / 8), d = (u - r * (D / 8)) * 8;
        const int rr = row0 + r, qi = rr / a.ratio, head = kvh * a.ratio + rr % a.ratio;
        if (qi >= nq) continue;
        float top_all = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top_all = fmaxf(top_all, xml[2 * (w * ROWS + r)]);
        float sum = 0.f, o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float tw = xml[2 * (w * ROWS + r)];
            if (tw == -INFINITY) continue;
            const float f = exp2f(tw - top_all);
            sum = fmaf(xml[2 * (w * ROWS + r) + 1], f, sum);
            const float* p = xs + (w * ROWS + r) * D + d;
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = fmaf(p[k], f, o[k]);
        }
        const int64_t row = static_cast<int64_t>(b) * a.seq + qi;
        if (a.splits > 1) {
            const int64_t at = (static_cast<int64_t>(split) * a.batch * a.seq + row) * a.nhead + head;
            if (d == 0) {
                a.part_ml[2 * at] = top_all;
                a.part_ml[2 * at + 1] = sum;
            }
            float4* p = reinterpret_cast<float4*>(a.part + at * D + d);
            p[0] = make_float4(o[0], o[1], o[2], o[3]);
            p[1] = make_float4(o[4], o[5], o[6], o[7]);
        } else if (d < a.c.dh[1]) {
            const float inv = top_all == -INFINITY ? 0.f : 1.f / sum;
            uint4 z;
            z.x = pack_half2(o[0] * inv, o[1] * inv);
            z.y = pack_half2(o[2] * inv, o[3] * inv);
            z.z = pack_half2(o[4] * inv, o[5] * inv);
            z.w = pack_half2(o[6] * inv, o[7] * inv);
            *reinterpret_cast<uint4*>(a.Z + row * a.ldz + head * a.c.dh[1] + d) = z;
        }
    }
}

// Joins the splits' partial results: a warp per (row, head), four features per lane.
__global__ void __launch_bounds__(128) attention_kv4_join_kernel(const AttArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t all = static_cast<int64_t>(a.batch) * a.seq * a.nhead;
    if (at >= all) return;
    const int64_t row = at / a.nhead;
    const int head = static_cast<int>(at - row * a.nhead), b = static_cast<int>(row / a.seq);
    const int qi = static_cast<int>(row - static_cast<int64_t>(b) * a.seq);
    if (a.q_len && qi >= __ldcg(a.q_len + b)) return;
    const int lane = threadIdx.x & 31, D = 32 * a.c.ng;
    // splits <= 64: two references per lane
    float t0 = lane < a.splits ? __ldcg(a.part_ml + 2 * (lane * all + at)) : -INFINITY;
    float t1 = lane + 32 < a.splits ? __ldcg(a.part_ml + 2 * ((lane + 32) * all + at)) : -INFINITY;
    float top = fmaxf(t0, t1);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    t0 = t0 == -INFINITY ? 0.f : exp2f(t0 - top);
    t1 = t1 == -INFINITY ? 0.f : exp2f(t1 - top);
    float sum = (lane < a.splits ? __ldcg(a.part_ml + 2 * (lane * all + at) + 1) * t0 : 0.f) +
                (lane + 32 < a.splits ? __ldcg(a.part_ml + 2 * ((lane + 32) * all + at) + 1) * t1 : 0.f);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < a.splits; ++s) {
        const float f = __shfl_sync(0xffffffffu, s < 32 ? t0 : t1, s & 31);
        if (f != 0.f && 4 * lane < D) {  // (f = 0 also where the split saw nothing; NaN passes)
            const float4 v = __ldcg(reinterpret_cast<const float4*>(a.part + (s * all + at) * D) + lane);
            o.x = fmaf(v.x, f, o.x);
            o.y = fmaf(v.y, f, o.y);
            o.z = fmaf(v.z, f, o.z);
            o.w = fmaf(v.w, f, o.w);
        }
    }
    if (4 * lane < a.c.dh[1]) {
        const float inv = top == -INFINITY ? 0.f : 1.f / sum;
        uint2 z;
        z.x = pack_half2(o.x * inv, o.y * inv);
        z.y = pack_half2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(a.Z + row * a.ldz + head * a.c.dh[1] + 4 * lane) = z;
    }
}

// Thread blocks along the sequence: enough for two to an SM, each with at least two tiles per warp.
int pick_splits(int64_t blocks, int max_len) {
    const int sms = sm_count() > 0 ? sm_count() : 148;
    int64_t s = (2 * sms + blocks - 1) / blocks;
    const int64_t most = (max_len + 2 * WARPS * TILE - 1) / (2 * WARPS * TILE);
    s = s < most ? s : most;
    return static_cast<int>(s < 1 ? 1 : (s > MAX_SPLITS ? MAX_SPLITS : s));
}

struct AttPlan {
    int rt, tiles, splits;
    size_t part, ml;
};
AttPlan plan_att(const Kv4View& v, int batch, int seq, int nhead, int max_len) {
    AttPlan p;
    const int64_t rows = static_cast<int64_t>(seq) * (nhead / v.nkv);
    p.rt = rows > 8 ? 2 : 1;
    p.tiles = static_cast<int>((rows + 8 * p.rt - 1) / (8 * p.rt));
    p.splits = pick_splits(static_cast<int64_t>(p.tiles) * v.nkv * batch, max_len);
    const size_t all = static_cast<size_t>(batch) * seq * nhead;
    p.part = p.splits > 1 ? p.splits * all * 32 * v.ng * sizeof(float) : 0;
    p.ml = p.splits > 1 ? p.splits * all * 2 * sizeof(float) : 0;
    return p;
}

template <int NG, int RT>
int launch_att(const AttArgs& a, cudaStream_t stream) {
    auto kern = attention_kv4_kernel<NG, RT>;
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !attr_set[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<NG>::TOTAL) != cudaSuccess)
            return ET_ERR_CUDA;
        attr_set[dev] = true;
    }
    const dim3 grid(a.splits, a.tiles * a.c.nkv, a.batch);
    return launch_kernel(kern, grid, dim3(THREADS), Smem<NG>::TOTAL, stream, a) == cudaSuccess ? ET_OK : ET_ERR_CUDA;
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
    if (!(scale > 0.f) || !(scale < INFINITY)) return ET_ERR_INVALID_ARG;
    if (static_cast<int64_t>(table_ld) << a.c.page_shift < max_len) return ET_ERR_SHAPE;
    if (ldq % 8 || ldz % 8 || ldq < static_cast<int64_t>(nhead) * a.c.dh[0] || ldz < static_cast<int64_t>(nhead) * a.c.dh[1])
        return ET_ERR_SHAPE;
    if (!et::aligned16(Q) || !et::aligned16(Z)) return ET_ERR_ALIGNMENT;
    const et::AttPlan p = et::plan_att(a.c, batch, seq, nhead, max_len);
    if (p.splits > 1) {
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
    a.rows = seq * a.ratio;
    a.tiles = p.tiles;
    a.splits = p.splits;
    a.scale_log2 = scale * et::LOG2E * 0x1p24f;
    a.err_word = et::device_error_word();
    if (!a.err_word) return ET_ERR_NO_DEVICE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (a.c.ng * 2 + p.rt) {
        case 3: st = et::launch_att<1, 1>(a, s); break;
        case 4: st = et::launch_att<1, 2>(a, s); break;
        case 5: st = et::launch_att<2, 1>(a, s); break;
        case 6: st = et::launch_att<2, 2>(a, s); break;
        case 7: st = et::launch_att<3, 1>(a, s); break;
        case 8: st = et::launch_att<3, 2>(a, s); break;
        case 9: st = et::launch_att<4, 1>(a, s); break;
        default: st = et::launch_att<4, 2>(a, s); break;
    }
    if (st != ET_OK || p.splits == 1) return st;
    const int64_t all = static_cast<int64_t>(batch) * seq * nhead;
    return et::launch_kernel(et::attention_kv4_join_kernel, dim3(static_cast<unsigned>((all + 3) / 4)), dim3(128), 0, s,
                             a) == cudaSuccess
               ? ET_OK
               : ET_ERR_CUDA;
}

}  // extern "C"
