// What the kernels of the 4-bit key/value cache share: the cache as they see it, and its argument checks.
#pragma once

#include "common.cuh"

#if defined(__CUDACC__)
#define KV4_HD __host__ __device__ __forceinline__
#else
#define KV4_HD inline
#endif

namespace et {

struct Kv4View {
    uint8_t* codes[2];  // K, V
    __half* params[2];
    int num_pages, page_shift, nkv, ng;
    int dh[2];
};

// ET_OK and `v` filled in, or a status.  Pointers are checked when `pointers` is set.
inline int kv4_view(const et_kv4_t* c, Kv4View& v, bool pointers) {
    if (!c || c->num_pages <= 0 || c->page <= 0 || c->nkv <= 0 || c->dh_qk <= 0 || c->dh_v <= 0)
        return ET_ERR_INVALID_ARG;
    if (c->page < 16 || (c->page & (c->page - 1)) || c->dh_qk % 16 || c->dh_v % 16 || c->dh_qk > 128 || c->dh_v > 128)
        return ET_ERR_SHAPE;
    if (static_cast<int64_t>(c->nkv) * 128 > INT32_MAX / 4) return ET_ERR_SHAPE;
    if (pointers) {
        if (!c->k_codes || !c->k_params || !c->v_codes || !c->v_params) return ET_ERR_INVALID_ARG;
        if (!aligned16(c->k_codes) || !aligned16(c->k_params) || !aligned16(c->v_codes) || !aligned16(c->v_params))
            return ET_ERR_ALIGNMENT;
    }
    v.codes[0] = c->k_codes;
    v.codes[1] = c->v_codes;
    v.params[0] = reinterpret_cast<__half*>(c->k_params);
    v.params[1] = reinterpret_cast<__half*>(c->v_params);
    v.num_pages = c->num_pages;
    v.page_shift = 0;
    while ((1 << v.page_shift) < c->page) ++v.page_shift;
    if (static_cast<int64_t>(c->num_pages) * c->nkv > INT64_MAX >> (v.page_shift + 8)) return ET_ERR_SHAPE;  // (bytes)
    v.nkv = c->nkv;
    v.dh[0] = c->dh_qk;
    v.dh[1] = c->dh_v;
    v.ng = ((c->dh_qk > c->dh_v ? c->dh_qk : c->dh_v) + 31) / 32;
    return ET_OK;
}

// x / d for 0 <= x < 2^31 by a multiplication
struct FastDiv {
    uint32_t mul, shift, d;
    FastDiv() = default;
    explicit FastDiv(uint32_t d_) : d(d_) {
        shift = 0;
        while ((1u << shift) < d && shift < 31) ++shift;
        mul = static_cast<uint32_t>(((1ull << (31 + shift)) + d - 1) / d);
    }
    KV4_HD uint32_t div(uint32_t x) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(x) * mul) >> (31 + shift));
    }
};

// Sizes that the attention over the cache takes (its grid, and 32-bit counts of rows and positions).
inline int kv4_check_attention(const Kv4View& v, int batch, int seq, int nhead, int max_len) {
    if (batch <= 0 || seq <= 0 || nhead <= 0 || max_len <= 0) return ET_ERR_INVALID_ARG;
    if (nhead % v.nkv || batch > 65535) return ET_ERR_SHAPE;
    const int64_t rows = static_cast<int64_t>(seq) * (nhead / v.nkv);
    if (static_cast<int64_t>(batch) * seq > INT32_MAX || rows > INT32_MAX / 2 || (rows > 8 ? (rows + 15) / 16 : 1) * v.nkv > 65535 ||
        max_len > INT32_MAX - (1 << 20) || static_cast<int64_t>(batch) * seq * nhead > INT32_MAX)
        return ET_ERR_SHAPE;
    return ET_OK;
}

#if defined(__CUDACC__)
// Page that holds position `pos` of a sequence, or -1 where the table does not reach or names no page of the cache.
__host__ __device__ __forceinline__ int kv4_page(const Kv4View& c, const int* table_row, int table_ld, int64_t pos) {
    const int64_t entry = pos >> c.page_shift;
    if (pos < 0 || entry >= table_ld) return -1;
#ifdef __CUDA_ARCH__
    const int id = __ldcg(table_row + entry);  // an earlier kernel may have written it
#else
    const int id = table_row[entry];
#endif
    return id < 0 || id >= c.num_pages ? -1 : id;
}
// Row of position `pos` in page `id` for key/value head `head`: rows of codes are 16 ng bytes, of params 4 ng.
__host__ __device__ __forceinline__ int64_t kv4_row(const Kv4View& c, int id, int64_t pos, int head) {
    return ((static_cast<int64_t>(id) * c.nkv + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}
#endif

}  // namespace et
