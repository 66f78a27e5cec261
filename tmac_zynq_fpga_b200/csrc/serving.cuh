// serving.cuh -- what the operators of the batched decode step share: the
// element types of a paged cache, its addressing, and the argument checks.
//
// A paged cache is two pools of pages, k and v, each [n_pages][kv_heads]
// [page_size][head_dim]: the page_size rows of one (page, head) lie together,
// so a tile of keys is one block copy per page.  page_size is a power of two.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>

#include <atomic>
#include <type_traits>

namespace tmac {

constexpr int kMaxPage = 256;

// Elements are read and written as 32-bit floats; the store rounds to nearest even.
template <typename T>
struct Elem;
template <>
struct Elem<float> {
    static TMAC_DEV float load(const float* p) { return *p; }
    static TMAC_DEV void store(float* p, float v) { *p = v; }
};
template <>
struct Elem<__half> {
    static TMAC_DEV float load(const __half* p) { return __half2float(*p); }
    static TMAC_DEV void store(__half* p, float v) { *p = __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
    static TMAC_DEV float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static TMAC_DEV void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
};

// 16-bit elements as pairs, the first in the low half.
template <typename T>
TMAC_DEV uint32_t pack2(float lo, float hi)
{
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <typename T>
TMAC_DEV void unpack2(uint32_t pair, float& lo, float& hi)
{
    if constexpr (std::is_same_v<T, __half>) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
        lo = f.x;
        hi = f.y;
    } else {
        lo = __uint_as_float(pair << 16);
        hi = __uint_as_float(pair & 0xFFFF0000u);
    }
}

inline int type_bytes(int type)
{
    return type == TMAC_TYPE_F32 ? 4 : (type == TMAC_TYPE_F16 || type == TMAC_TYPE_BF16) ? 2 : 0;
}

// Calls f with a null pointer of the element type that `type` names.
template <typename F>
int with_type(int type, F&& f)
{
    switch (type) {
    case TMAC_TYPE_F32: return f((float*)nullptr);
    case TMAC_TYPE_F16: return f((__half*)nullptr);
    case TMAC_TYPE_BF16: return f((__nv_bfloat16*)nullptr);
    default: return fail(TMAC_ERR_TYPE, "element type must be F32, F16 or BF16");
    }
}

// The cache as a kernel sees it.
struct CacheDev {
    void *k, *v;
    int64_t n_pages;
    int kv_heads, page_shift, dim;
};

TMAC_DEV void record_error(int* err, int code) { atomicExch(err, code); }

// Kernel attributes are set once per kernel and device: `done` has a bit for each device.
template <typename F>
int set_once(std::atomic<uint64_t>& done, int device, F&& set)
{
    const uint64_t bit = 1ull << (device & 63);
    if (done.load(std::memory_order_acquire) & bit) return TMAC_OK;
    TMAC_CUDA_TRY(set());
    done.fetch_or(bit, std::memory_order_release);
    return TMAC_OK;
}

// Host-side checks, none of which touches a device.
inline int check_cache(const tmac_paged_cache* c, CacheDev* out)
{
    if (!c || !c->k || !c->v) return fail(TMAC_ERR_INVALID, "NULL cache");
    if (!type_bytes(c->type)) return fail(TMAC_ERR_TYPE, "cache type must be F32, F16 or BF16");
    if (c->n_pages <= 0 || c->n_pages > 0x7FFFFFFF || c->kv_heads <= 0 || c->kv_heads > 65535)
        return fail(TMAC_ERR_SHAPE, "cache needs pages and heads");
    if (c->page_size < 1 || c->page_size > kMaxPage || (c->page_size & (c->page_size - 1)))
        return fail(TMAC_ERR_SHAPE, "page_size must be a power of two up to 256");
    if (c->head_dim < 2 || c->head_dim > 1024 || c->head_dim % 2)
        return fail(TMAC_ERR_SHAPE, "head_dim must be even, 2 to 1024");
    if (c->device < 0) return fail(TMAC_ERR_NODEV, "no such CUDA device");
    if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16) return fail(TMAC_ERR_INVALID, "cache pools must be 16-byte aligned");
    out->k = c->k;
    out->v = c->v;
    out->n_pages = c->n_pages;
    out->kv_heads = c->kv_heads;
    out->page_shift = __builtin_ctz((unsigned)c->page_size);
    out->dim = c->head_dim;
    return TMAC_OK;
}

}  // namespace tmac
