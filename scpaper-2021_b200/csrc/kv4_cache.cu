// Writing fp16 keys and values into the 4-bit cache, and reading them back.
//
// Four lanes serve one (token, head) row of K or of V.  Lane j holds features 32 g + 8 j .. + 8 of every group g
// (16-byte loads and stores on the fp16 side), so a group's range is two shuffles over the four lanes, and in the
// cache the lane owns the 4 ng consecutive bytes of its features: one store or load per lane (K: word j of
// each group; V: units 2 j and 2 j + 1 of each group).  Lane g < ng also moves group g's (s, m).
//
// What bounds it: HBM (2 + 0.625 bytes a value each way).
#include "kernels.h"
#include "kv4.h"
#include "quant4.cuh"

namespace et {
namespace {

constexpr int KV_THREADS = 256;

struct Kv4Move {
    Kv4View c;
    __half* x[2];  // fp16 K and V
    int ld[2];
    const int* table;
    const int* start;
    const int* len;
    int table_ld, batch, seq;
    int rows_per_token;  // 2 nkv
    int64_t quads;       // rows in all
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

template <int NG, bool WRITE>
__global__ void __launch_bounds__(KV_THREADS) kv4_move_kernel(const Kv4Move a) {
    pdl_wait();
    pdl_launch_dependents();
    const int64_t q = (static_cast<int64_t>(blockIdx.x) * KV_THREADS + threadIdx.x) >> 2;
    const int j = threadIdx.x & 3;
    // (the lanes of a row leave together, those past the last row stay for the shuffles)
    const int token = q < a.quads ? static_cast<int>(q / a.rows_per_token) : 0;
    const int r = q < a.quads ? static_cast<int>(q - static_cast<int64_t>(token) * a.rows_per_token) : 0;
    const int b = token / a.seq, i = token - b * a.seq;
    const int of = r >= a.c.nkv ? 1 : 0, head = r - of * a.c.nkv;
    const int n = a.len ? __ldcg(a.len + b) : a.seq;
    bool live = q < a.quads && i < n;
    int64_t row = -1;
    if (live) {
        const int64_t pos = static_cast<int64_t>(a.start ? __ldcg(a.start + b) : 0) + i;
        const int id = kv4_page(a.c, a.table + static_cast<int64_t>(b) * a.table_ld, a.table_ld, pos);
        row = id < 0 ? -1 : kv4_row(a.c, id, pos, head);
        if (row < 0 && j == 0) atomicCAS(a.err_word, 0, DEV_BAD_PAGE);
    }
    const int dh = a.c.dh[of];
    __half* x = a.x[of] + static_cast<int64_t>(token) * a.ld[of] + head * dh + 8 * j;
    if (WRITE) {
        live = live && row >= 0;
        uint4 v[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            v[g] = make_uint4(0, 0, 0, 0);
            if (live && 32 * g + 8 * j < dh) v[g] = __ldcg(reinterpret_cast<const uint4*>(x + 32 * g));
        }
        uint32_t w[NG], sm_mine = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const bool in = 32 * g + 8 * j < dh;
            q4::Range range = {INFINITY, -INFINITY, true};
            if (in) range = q4::range8(v[g]);
            q4::range_quad(range);
            const uint32_t sm = 32 * g < dh ? q4::params_of(range) : 0u;
            w[g] = in ? q4::codes8(v[g], sm) : 0u;
            if (g == j) sm_mine = sm;
        }
        if (live) {
            uint32_t out[NG];
            if (of == 0) {
#pragma unroll
                for (int g = 0; g < NG; ++g) out[g] = q4::to_pairs(w[g]);
            } else {
                units_of_words<NG>(w, out);
            }
            store_words<NG>(a.c.codes[of] + row * (16 * NG) + j * (4 * NG), out);
            if (j < NG) reinterpret_cast<uint32_t*>(a.c.params[of])[row * NG + j] = sm_mine;
        }
    } else if (live) {
        uint32_t w[NG], sm[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) w[g] = sm[g] = 0u;
        if (row >= 0) {
            uint32_t raw[NG];
            load_words<NG>(a.c.codes[of] + row * (16 * NG) + j * (4 * NG), raw);
            load_words<NG>(reinterpret_cast<const uint8_t*>(a.c.params[of]) + row * (4 * NG), sm);
            if (of == 0) {
#pragma unroll
                for (int g = 0; g < NG; ++g) w[g] = q4::from_pairs(raw[g]);
            } else {
                words_of_units<NG>(raw, w);
            }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
            if (32 * g + 8 * j < dh) *reinterpret_cast<uint4*>(x + 32 * g) = q4::values8(w[g], sm[g]);
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
    a.rows_per_token = 2 * a.c.nkv;
    a.quads = static_cast<int64_t>(batch) * seq * a.rows_per_token;
    const int64_t blocks = (a.quads * 4 + KV_THREADS - 1) / KV_THREADS;
    if (blocks > INT32_MAX) return ET_ERR_SHAPE;
    a.err_word = device_error_word();
    if (!a.err_word) return ET_ERR_NO_DEVICE;
    void (*const kernels[4])(const Kv4Move) = {kv4_move_kernel<1, WRITE>, kv4_move_kernel<2, WRITE>,
                                               kv4_move_kernel<3, WRITE>, kv4_move_kernel<4, WRITE>};
    return launch_kernel(kernels[a.c.ng - 1], dim3(static_cast<unsigned>(blocks)), dim3(KV_THREADS), 0, stream, a) ==
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
