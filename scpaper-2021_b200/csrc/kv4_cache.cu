// Writing fp16 keys and values into the 4-bit cache, and reading them back.
//
// Four lanes serve the rows of one (token, head) in K and in V.  Lane j holds features 32 g + 8 j .. + 8 of every group
// g (16-byte loads and stores on the fp16 side), so a group's range is two shuffles over the four lanes, and in
// the cache the lane owns the 4 ng consecutive bytes of its features: one store or load per lane (K: word j of
// each group; V: units 2 j and 2 j + 1 of each group).  Lane g < ng also writes group g's (s, m).  A warp covers
// eight consecutive tokens of a head: its rows lie together in the cache (ng = 2: 256 bytes of codes, 64 of
// parameters), and a token's head is a whole line or more of the fp16 side anyway.
//
// What bounds it.  Reading: HBM (4 x 8191 tokens, 8 heads of 128: 30.1 us, 5.8 TB/s).  Writing: instruction issue, 18 per
// value and lane (8 x 2048 tokens, 16 heads of 64: about 28 us, 3.1 TB/s).  Registers are held down for more warps
// (write + read back of those: 44.9 us; 46.3 where the compiler chose, 57.2 where it took what it liked); several
// heads to a warp, the next one's values in flight, took 50.0.
#include "kernels.h"
#include "kv4.h"
#include "quant4.cuh"

namespace et {
namespace {

constexpr int KV_THREADS = 128;

struct Kv4Move {
    Kv4View c;
    __half* x[2];  // fp16 K and V
    int ld[2];
    const int* table;
    const int* start;
    const int* len;
    int table_ld, batch, seq, tokens;
    FastDiv by_heads, by_seq;
    int* err_word;
};

// The 4 ng bytes of one lane.
template <int NG>
__device__ __forceinline__ void store_words(uint8_t* p, const uint32_t (&w)[NG]) {
    if (NG == 4) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[NG > 1], w[NG > 2 ? 2 : 0], w[NG > 3 ? 3 : 0]);
    else if (NG == 2) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[NG > 1]);
    else
#pragma unroll
        for (int g = 0; g < NG; ++g) reinterpret_cast<uint32_t*>(p)[g] = w[g];
}
template <int NG>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[NG]) {
    if (NG == 4) {
        const uint4 v = __ldcg(reinterpret_cast<const uint4*>(p));
        w[0] = v.x, w[NG > 1] = v.y, w[NG > 2 ? 2 : 0] = v.z, w[NG > 3 ? 3 : 0] = v.w;
    } else if (NG == 2) {
        const uint2 v = __ldcg(reinterpret_cast<const uint2*>(p));
        w[0] = v.x, w[NG > 1] = v.y;
    } else {
#pragma unroll
        for (int g = 0; g < NG; ++g) w[g] = __ldcg(reinterpret_cast<const uint32_t*>(p) + g);
    }
}
// V: lane words (features 8 j .. + 8 of each group, natural nibble order) <-> units [2 j][ng], [2 j + 1][ng]
template <int NG>
__device__ __forceinline__ void units_of_words(const uint32_t (&w)[NG], uint32_t (&u)[NG]) {
#pragma unroll
    for (int k = 0; k < NG; ++k) {  // word k of the result: units 2 k and 2 k + 1 of the 2 NG
        const int a = 2 * k, b = 2 * k + 1;
        u[k] = __byte_perm(w[a % NG], w[b % NG], (a / NG ? 0x0032 : 0x0010) | (b / NG ? 0x7600 : 0x5400));
    }
}
template <int NG>
__device__ __forceinline__ void words_of_units(const uint32_t (&u)[NG], uint32_t (&w)[NG]) {
#pragma unroll
    for (int g = 0; g < NG; ++g) {  // units g (low half) and NG + g (high half)
        const int a = g, b = NG + g;
        w[g] = __byte_perm(u[a / 2], u[b / 2], (a & 1 ? 0x0032 : 0x0010) | (b & 1 ? 0x7600 : 0x5400));
    }
}

// FULL: both heads are 32 NG features wide.
template <int NG, bool WRITE, bool FULL>
__global__ void __launch_bounds__(KV_THREADS, NG <= 2 ? 12 : (NG == 3 ? 8 : 6)) kv4_move_kernel(const Kv4Move a) {
    const int dh[2] = {FULL ? 32 * NG : a.c.dh[0], FULL ? 32 * NG : a.c.dh[1]};
    auto inside = [&](int of, int first) { return FULL || first < dh[of]; };  // a feature of the head
    pdl_wait();
    pdl_launch_dependents();
    // unit: (eight tokens, head, token of the eight), four lanes each
    const uint32_t unit = blockIdx.x * (KV_THREADS / 32) + (threadIdx.x >> 5);
    const uint32_t eight = a.by_heads.div(unit);
    const int head = static_cast<int>(unit - eight * a.by_heads.d);
    const int lane = threadIdx.x & 31, j = lane & 3;
    const int64_t token = static_cast<int64_t>(eight) * 8 + (lane >> 2);
    bool live = token < a.tokens;  // (the lanes that are not stay for the shuffles)
    const int b = static_cast<int>(a.by_seq.div(live ? static_cast<uint32_t>(token) : 0u));
    const int i = static_cast<int>(token) - b * a.seq;
    live = live && i < (a.len ? __ldcg(a.len + b) : a.seq);
    uint4 v[2][NG];
    __half* x[2];
#pragma unroll
    for (int of = 0; of < 2; ++of) {
        x[of] = a.x[of] + token * a.ld[of] + head * dh[of] + 8 * j;
        if (WRITE)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                v[of][g] = make_uint4(0, 0, 0, 0);
                if (live && inside(of, 32 * g + 8 * j))
                    v[of][g] = __ldcg(reinterpret_cast<const uint4*>(x[of] + 32 * g));
            }
    }
    int64_t row = -1;
    if (live) {
        const int64_t pos = static_cast<int64_t>(a.start ? __ldcg(a.start + b) : 0) + i;
        const int id = kv4_page(a.c, a.table + static_cast<int64_t>(b) * a.table_ld, a.table_ld, pos);
        row = id < 0 ? -1 : kv4_row(a.c, id, pos, head);
        if (row < 0 && j == 0) atomicCAS(a.err_word, 0, DEV_BAD_PAGE);
    }
    const bool there = live && row >= 0;
    uint32_t raw[2][NG], sm[2][NG];
    if (!WRITE) {
#pragma unroll
        for (int of = 0; of < 2; ++of) {
#pragma unroll
            for (int g = 0; g < NG; ++g) raw[of][g] = sm[of][g] = 0u;
            if (there) {
                load_words<NG>(a.c.codes[of] + row * (16 * NG) + j * (4 * NG), raw[of]);
                load_words<NG>(reinterpret_cast<const uint8_t*>(a.c.params[of]) + row * (4 * NG), sm[of]);
            }
        }
    }
    float inv[2][NG];
    if (WRITE) {
        // The lanes of a row share the ranges out: after two exchanges lane j holds the whole range of every fourth
        // (tensor, group), makes its (s, m) and 1 / s, and the others fetch them.
        constexpr int N = (2 * NG + 3) / 4 * 4;
        uint32_t r[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int of = k / NG, g = k % NG;
            r[k] = k < 2 * NG && inside(of & 1, 32 * g + 8 * j) ? q4::range8(v[of & 1][g]) : q4::EMPTY_RANGE;
        }
#pragma unroll
        for (int k = 0; k < N; k += 4) {
            const bool one = (j & 1) != 0, two = (j & 2) != 0;
            const uint32_t lo = q4::range_join(one ? r[k + 1] : r[k],
                                               __shfl_xor_sync(0xffffffffu, one ? r[k] : r[k + 1], 1));
            const uint32_t hi = q4::range_join(one ? r[k + 3] : r[k + 2],
                                               __shfl_xor_sync(0xffffffffu, one ? r[k + 2] : r[k + 3], 1));
            const uint32_t mine = q4::range_join(two ? hi : lo, __shfl_xor_sync(0xffffffffu, two ? lo : hi, 2));
            const uint32_t p = (!FULL || k + 4 > 2 * NG) && mine == q4::EMPTY_RANGE ? 0u : q4::params_of(mine);
            const float i1 = q4::inverse_of(p);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (k + q < 2 * NG) {
                    const int of = (k + q) / NG, g = (k + q) % NG;
                    sm[of][g] = __shfl_sync(0xffffffffu, p, q, 4);
                    inv[of][g] = __shfl_sync(0xffffffffu, i1, q, 4);
                }
        }
    }
#pragma unroll
    for (int of = 0; of < 2; ++of) {
        uint32_t w[NG];
        if (WRITE) {
            uint32_t mine = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t c = of == 0 ? q4::codes8<true>(v[of][g], sm[of][g], inv[of][g])
                                           : q4::codes8<false>(v[of][g], sm[of][g], inv[of][g]);
                w[g] = inside(of, 32 * g + 8 * j) ? c : 0u;
                if (g == j) mine = sm[of][g];
            }
            if (there) {
                uint32_t out[NG];
                if (of == 0) {
#pragma unroll
                    for (int g = 0; g < NG; ++g) out[g] = w[g];
                } else {
                    units_of_words<NG>(w, out);
                }
                store_words<NG>(a.c.codes[of] + row * (16 * NG) + j * (4 * NG), out);
                if (j < NG) reinterpret_cast<uint32_t*>(a.c.params[of])[row * NG + j] = mine;
            }
        } else if (live) {
            if (of == 0) {
#pragma unroll
                for (int g = 0; g < NG; ++g) w[g] = raw[of][g];
            } else {
                words_of_units<NG>(raw[of], w);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (inside(of, 32 * g + 8 * j))
                    *reinterpret_cast<uint4*>(x[of] + 32 * g) =
                        of == 0 ? q4::values8<true>(w[g], sm[of][g]) : q4::values8<false>(w[g], sm[of][g]);
        }
    }
}

template <bool WRITE>
int move(const et_kv4_t* cache, __half* K, __half* V, int ldk, int ldv, const int32_t* table, int table_ld,
         const int32_t* start, const int32_t* len, int batch, int seq, cudaStream_t stream) {
    Kv4Move a = {};
    const int st = kv4_view(cache, a.c, true);
    if (st != ET_OK) return st;
    if (!K || !V || !table || table_ld <= 0 || batch <= 0 || seq <= 0) return ET_ERR_INVALID_ARG;
    if (ldk % 8 || ldv % 8 || ldk < a.c.nkv * a.c.dh[0] || ldv < a.c.nkv * a.c.dh[1]) return ET_ERR_SHAPE;
    if (static_cast<int64_t>(batch) * seq > INT32_MAX) return ET_ERR_SHAPE;
    if (!aligned16(K) || !aligned16(V)) return ET_ERR_ALIGNMENT;
    a.x[0] = K, a.x[1] = V;
    a.ld[0] = ldk, a.ld[1] = ldv;
    a.table = table, a.start = start, a.len = len;
    a.table_ld = table_ld, a.batch = batch, a.seq = seq;
    a.tokens = batch * seq;
    a.by_heads = FastDiv(static_cast<uint32_t>(a.c.nkv));
    a.by_seq = FastDiv(static_cast<uint32_t>(seq));
    const int64_t units = (static_cast<int64_t>(a.tokens) + 7) / 8 * a.c.nkv;
    if (units > INT32_MAX - KV_THREADS) return ET_ERR_SHAPE;
    const int64_t blocks = (units + KV_THREADS / 32 - 1) / (KV_THREADS / 32);
    a.err_word = device_error_word();
    if (!a.err_word) return ET_ERR_NO_DEVICE;
    void (*const kernels[8])(const Kv4Move) = {
        kv4_move_kernel<1, WRITE, false>, kv4_move_kernel<2, WRITE, false>, kv4_move_kernel<3, WRITE, false>,
        kv4_move_kernel<4, WRITE, false>, kv4_move_kernel<1, WRITE, true>,  kv4_move_kernel<2, WRITE, true>,
        kv4_move_kernel<3, WRITE, true>,  kv4_move_kernel<4, WRITE, true>};
    const bool full = a.c.dh[0] == 32 * a.c.ng && a.c.dh[1] == 32 * a.c.ng;
    return launch_kernel(kernels[a.c.ng - 1 + (full ? 4 : 0)], dim3(static_cast<unsigned>(blocks)), dim3(KV_THREADS), 0, stream, a) ==
                   cudaSuccess
               ? ET_OK
               : ET_ERR_CUDA;
}

}  // namespace
}  // namespace et

extern "C" {

#ifdef ET_TEST_HOOKS
// Test hook: the row of a position as the kernels find it, from a table in host memory; -1: none.
long long et_debug_kv4_row(const et_kv4_t* cache, const int32_t* table_row, int table_ld, long long pos, int head) {
    et::Kv4View v;
    if (et::kv4_view(cache, v, false) != ET_OK) return -2;
    const int id = et::kv4_page(v, table_row, table_ld, pos);
    return id < 0 ? -1 : et::kv4_row(v, id, pos, head);
}
#endif  // ET_TEST_HOOKS

int et_kv4_sizes(const et_kv4_t* cache, size_t* code_bytes, size_t* param_bytes) {
    et::Kv4View v;
    if (!code_bytes || !param_bytes) return ET_ERR_INVALID_ARG;
    const int st = et::kv4_view(cache, v, false);
    if (st != ET_OK) return st;
    const size_t rows = (static_cast<size_t>(v.num_pages) * v.nkv) << v.page_shift;
    *code_bytes = rows * 16 * v.ng;
    *param_bytes = rows * 4 * v.ng;
    return ET_OK;
}

int et_kv4_write_fwd(const et_kv4_t* cache, const et_half* K, const et_half* V, int ldk, int ldv,
                     const int32_t* table, int table_ld, const int32_t* start, const int32_t* new_len, int batch,
                     int seq, et_stream stream) {
    return et::move<true>(cache, reinterpret_cast<__half*>(const_cast<et_half*>(K)),
                          reinterpret_cast<__half*>(const_cast<et_half*>(V)), ldk, ldv, table, table_ld, start,
                          new_len, batch, seq, static_cast<cudaStream_t>(stream));
}

int et_kv4_read_fwd(const et_kv4_t* cache, et_half* K, et_half* V, int ldk, int ldv, const int32_t* table,
                    int table_ld, const int32_t* start, const int32_t* len, int batch, int seq, et_stream stream) {
    return et::move<false>(cache, reinterpret_cast<__half*>(K), reinterpret_cast<__half*>(V), ldk, ldv, table,
                           table_ld, start, len, batch, seq, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
