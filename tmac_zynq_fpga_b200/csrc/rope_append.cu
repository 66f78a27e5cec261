// rope_append.cu -- q, k and v of a step: bias, position rotation, and k and v
// stored into a paged cache (bias + apply_rope + cache writes of
// forward_layer_with_cache, sim/tmac_gguf.cpp:1528-1554, :1590-1622, for a batch of
// tokens of several sequences).
//
// For pair i of a head, with c = cos[pos][i], s = sin[pos][i]:
//   (a, z) -> (a c - z s, a s + z c),
// pairs (2i, 2i + 1) when interleaved, else (i, i + rot_dim / 2); the values past
// rot_dim pass through.  Products and sums are 32-bit, each rounded by itself as in the
// reference, and the result once to the cache's type.
//
// Bound: HBM, every value is read once and written once (32768 tokens of 16/4 heads of
// 128, bf16, 92.5 us, 4490 GB/s; 512 tokens 3.6 us, 2 tokens 3.3, the launch).  Where
// the pointers, strides and head parts allow it a thread takes 8 adjoining values (16
// bytes of a 16-bit type), or 8 pairs of halves, and keeps that place in a token for all
// tokens of its CTA, the next one's values loaded beneath the work on this one's: 16-bit
// values 98 -> 91 us and 21.3 -> 19.3 against places dealt out anew, 32-bit ones 34 ->
// 36.6, 49 -> 50 and, of 512 tokens, 3.9 -> 3.5 (then with fused multiply-adds, 1 to 2 %
// faster, but rounding otherwise than the other kernel).  A CTA first looks up its tokens' pages,
// cosines and sines into shared memory, so nothing but the values is waited for.  Other
// layouts take one pair per thread.
#include "serving.cuh"

#include <algorithm>

namespace tmac {
namespace {

// (a, z) by cosine c and sine s; every kernel rounds the same, whatever the layout.
TMAC_DEV void rotate(float& a, float& z, float c, float s)
{
    const float x = __fadd_rn(__fmul_rn(a, c), -__fmul_rn(z, s));
    z = __fadd_rn(__fmul_rn(a, s), __fmul_rn(z, c));
    a = x;
}

struct RopeArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements between tokens
    void* q_out;
    const float* bias;
    const int *seq, *pos, *starts, *tables;
    const float *cos, *sin;
    int64_t tokens;
    int heads, n_seq, table_width, max_pos, rot;
    CacheDev cache;
    int* err;
};

// Where token t goes.  ok: its row is computed; page < 0: it is not stored.
struct Place {
    bool ok;
    int pos, slot;
    int64_t page;
};
TMAC_DEV Place place_of(const RopeArgs& a, int64_t t)
{
    Place p = {false, 0, 0, -1};
    const int seq = a.seq ? a.seq[t] : (int)t;
    if (seq < 0) return p;  // padding
    p.pos = a.pos[t];
    if (seq >= a.n_seq || p.pos < 0 || p.pos >= a.max_pos) {
        record_error(a.err, TMAC_ERR_BOUNDS);
        return p;
    }
    p.ok = true;
    const int own = p.pos - (a.starts ? a.starts[seq] : 0);
    const int shift = a.cache.page_shift;
    if (own >= 0 && (own >> shift) < a.table_width) {
        p.page = a.tables[(int64_t)seq * a.table_width + (own >> shift)];
        p.slot = own & ((1 << shift) - 1);
    }
    if (p.page < 0 || p.page >= a.cache.n_pages) {
        p.page = -1;
        record_error(a.err, TMAC_ERR_BOUNDS);
    }
    return p;
}

// One pair of values per thread.
template <typename T, typename C, bool kInterleaved>
__global__ void __launch_bounds__(256) rope_append_kernel(RopeArgs a)
{
    const int d = a.cache.dim, pairs = d / 2, hk = a.cache.kv_heads;
    const int per_token = (a.heads + 2 * hk) * pairs;
    const int64_t n = a.tokens * per_token;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t t = i / per_token;
        const int u = (int)(i - t * per_token);
        const int row = u / pairs, pair = u - row * pairs;
        const bool is_q = row < a.heads, is_v = row >= a.heads + hk;
        const int head = is_q ? row : is_v ? row - a.heads - hk : row - a.heads;
        // the pair's two values within the head, and whether they are rotated
        int d0 = 2 * pair, d1 = 2 * pair + 1;
        const bool turn = !is_v && 2 * pair < a.rot;
        if (!kInterleaved && turn) {
            d0 = pair;
            d1 = pair + a.rot / 2;
        }
        const T* src = is_q   ? (const T*)a.q + t * a.q_stride
                       : is_v ? (const T*)a.v + t * a.v_stride
                              : (const T*)a.k + t * a.k_stride;
        src += (int64_t)head * d;
        const Place p = place_of(a, t);
        C* dst;
        if (is_q)
            dst = (C*)a.q_out + (t * a.heads + head) * d;
        else if (p.page >= 0)
            dst = (C*)(is_v ? a.cache.v : a.cache.k) + (((p.page * hk + head) << a.cache.page_shift) + p.slot) * d;
        else
            continue;
        float x = 0.0f, z = 0.0f;
        if (p.ok) {
            x = Elem<T>::load(src + d0);
            z = Elem<T>::load(src + d1);
            if (a.bias) {
                x = __fadd_rn(x, a.bias[(int64_t)row * d + d0]);
                z = __fadd_rn(z, a.bias[(int64_t)row * d + d1]);
            }
            if (turn) {
                rotate(x, z, a.cos[(int64_t)p.pos * (a.rot / 2) + pair], a.sin[(int64_t)p.pos * (a.rot / 2) + pair]);
            }
        }
        Elem<C>::store(dst + d0, x);
        Elem<C>::store(dst + d1, z);
    }
}

// 8 adjoining elements, as they lie and as floats.
template <typename T>
struct Eight {
    uint4 raw[sizeof(T) / 2];
    TMAC_DEV void load(const T* p)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
    TMAC_DEV void floats(float (&x)[8]) const
    {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) unpack2<T>(w[i], x[2 * i], x[2 * i + 1]);
        }
    }
    TMAC_DEV void set(const float (&x)[8])
    {
        uint32_t* w = reinterpret_cast<uint32_t*>(raw);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = __float_as_uint(x[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
        }
    }
};
template <typename T>
TMAC_DEV void store8(T* p, const float (&x)[8])
{
    Eight<T> e;
    e.set(x);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4*>(p)[i] = e.raw[i];
}
TMAC_DEV void add8(float (&x)[8], const float* bias)
{
    Eight<float> e;
    e.load(bias);
    float b[8];
    e.floats(b);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __fadd_rn(x[i], b[i]);
}

// Division of a number below 2^16 by a fixed one below 2^16.
struct Divide {
    uint32_t by, magic;
    static Divide of(int by) { return {(uint32_t)by, (uint32_t)((0x100000000ull + by - 1) / by)}; }
    TMAC_DEV int operator()(int x) const { return by == 1 ? x : (int)__umulhi((uint32_t)x, magic); }
};
// Units of a q or k head: 8 values at a time (interleaved), or 8 pairs at a time of
// the rotated part and 8 values at a time of the rest; of a v head: 8 values at a time.
constexpr int kMaxTokens = 16;  // of a CTA
template <typename T>
constexpr int kMaxThreads = sizeof(T) == 2 ? 512 : 384;  // 32-bit values take more registers
struct Deal {
    int tokens;     // of a CTA
    int units;      // of a token
    int turned;     // of these, of q and k heads
    Divide per_head, per_v;
};
template <typename T, typename C, bool kInterleaved>
__global__ void __launch_bounds__(kMaxThreads<T>, sizeof(T) == 2 ? 2 : 1) rope_append_vec_kernel(RopeArgs a, Deal deal)
{
    extern __shared__ __align__(16) float turns[];  // [tokens][2][rot / 2]: cosines, sines
    __shared__ Place places[kMaxTokens];
    const int d = a.cache.dim, hk = a.cache.kv_heads, shift = a.cache.page_shift, half = a.rot / 2;
    const int pairs8 = kInterleaved ? 0 : a.rot / 16;
    const int64_t t0 = (int64_t)blockIdx.x * deal.tokens;
    const int n = (int)min((int64_t)deal.tokens, a.tokens - t0);
    // a thread keeps its unit for all tokens of the CTA
    bool is_v, halves;
    int row, d0;  // row: of q, k and v together
    const T* src;
    int64_t stride;
    const auto take = [&](int u) {
        is_v = u >= deal.turned;
        if (is_v) {
            u -= deal.turned;
            const int head = deal.per_v(u);
            row = a.heads + hk + head;
            d0 = (u - head * (int)deal.per_v.by) * 8;
            halves = false;
            src = (const T*)a.v + head * d;
            stride = a.v_stride;
        } else {
            row = deal.per_head(u);
            const int unit = u - row * (int)deal.per_head.by;
            halves = unit < pairs8;
            d0 = halves || kInterleaved ? unit * 8 : a.rot + (unit - pairs8) * 8;
            const bool is_k = row >= a.heads;
            src = is_k ? (const T*)a.k + (row - a.heads) * d : (const T*)a.q + row * d;
            stride = is_k ? a.k_stride : a.q_stride;
        }
        src += t0 * stride + d0;
    };
    Eight<T> xr, zr;
    const auto load = [&] {
        xr.load(src);
        if (halves) zr.load(src + half);
        src += stride;
    };
    int u = threadIdx.x;
    if (u < deal.units) {
        take(u);
        load();
    }
    if ((int)threadIdx.x < n) places[threadIdx.x] = place_of(a, t0 + threadIdx.x);
    __syncthreads();
    for (int i = threadIdx.x; i < n * (a.rot / 4); i += blockDim.x) {
        const int token = i / (a.rot / 4), at = i % (a.rot / 4) * 4;  // of cosines, then of sines
        if (!places[token].ok) continue;
        const float* from = (at < half ? a.cos + at : a.sin + at - half) + (int64_t)places[token].pos * half;
        *reinterpret_cast<float4*>(turns + token * a.rot + at) = __ldg(reinterpret_cast<const float4*>(from));
    }
    __syncthreads();
    while (u < deal.units) {
        const bool is_q = row < a.heads;
        // q's row of the first token; of k and v the place in a page
        C* const to = is_q ? (C*)a.q_out + (t0 * a.heads + row) * d + d0
                           : (C*)(is_v ? a.cache.v : a.cache.k) + ((int64_t)(row - a.heads - (is_v ? hk : 0)) << shift) * d + d0;
        for (int token = 0; token < n; token++) {
            float x[8], z[8];
            xr.floats(x);
            if (halves) zr.floats(z);
            if (token + 1 < n) load();  // beneath this token's arithmetic
            const Place& p = places[token];
            C* dst = to;
            if (is_q)
                dst += (int64_t)token * (a.heads * d);
            else if (p.page >= 0)
                dst += (((p.page * hk) << shift) + p.slot) * d;
            else
                continue;
            if (a.bias) {
                add8(x, a.bias + row * d + d0);
                if (halves) add8(z, a.bias + row * d + d0 + half);
            }
            const float *c = turns + token * a.rot, *s = c + half;
            if (!p.ok) {
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = z[i] = 0.0f;
            } else if (kInterleaved && !is_v && d0 < a.rot) {
                const float4 c4 = *reinterpret_cast<const float4*>(c + d0 / 2), s4 = *reinterpret_cast<const float4*>(s + d0 / 2);
                const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int i = 0; i < 4; i++) rotate(x[2 * i], x[2 * i + 1], cv[i], sv[i]);
            } else if (halves) {
#pragma unroll
                for (int h = 0; h < 8; h += 4) {
                    const float4 c4 = *reinterpret_cast<const float4*>(c + d0 + h), s4 = *reinterpret_cast<const float4*>(s + d0 + h);
                    const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) rotate(x[h + i], z[h + i], cv[i], sv[i]);
                }
            }
            store8(dst, x);
            if (halves) store8(dst + half, z);
        }
        u += blockDim.x;
        if (u < deal.units) {
            take(u);
            load();
        }
    }
}

// Whether the 16-byte accesses of the vector kernel are aligned.
template <typename T, typename C>
bool vectors_fit(const RopeArgs& a, bool interleaved)
{
    auto aligned = [](const void* p) { return (uintptr_t)p % 16 == 0; };
    const int64_t vec = 16 / (int64_t)sizeof(T);
    return a.cache.dim % 8 == 0 && a.cache.dim <= 256 && a.rot % (interleaved ? 8 : 16) == 0 && aligned(a.q) && aligned(a.k) && aligned(a.v) &&
           a.q_stride % vec == 0 && a.k_stride % vec == 0 && a.v_stride % vec == 0 && aligned(a.q_out) &&
           aligned(a.bias) && aligned(a.cos) && aligned(a.sin);
}

template <typename T, typename C>
int launch_rope(const RopeArgs& a, bool interleaved, int sms, cudaStream_t s)
{
    const int hk = a.cache.kv_heads, per_head = interleaved ? a.cache.dim / 8 : a.rot / 16 + (a.cache.dim - a.rot) / 8;
    const int64_t per_token = (int64_t)(a.heads + hk) * per_head + hk * (a.cache.dim / 8);
    if (per_token < 4096 && vectors_fit<T, C>(a, interleaved)) {
        Deal d;
        // tokens of a CTA: as long as there are four CTAs to an SM
        d.tokens = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxTokens, a.tokens / (4 * sms)));
        d.units = (int)per_token;
        d.turned = (a.heads + hk) * per_head;
        d.per_head = Divide::of(per_head);
        d.per_v = Divide::of(a.cache.dim / 8);
        // threads: a token's units, or an even part of them
        const int parts = (d.units + kMaxThreads<T> - 1) / kMaxThreads<T>, threads = ((d.units + parts - 1) / parts + 31) / 32 * 32;
        auto fn = interleaved ? rope_append_vec_kernel<T, C, true> : rope_append_vec_kernel<T, C, false>;
        fn<<<(unsigned)((a.tokens + d.tokens - 1) / d.tokens), threads, (size_t)d.tokens * a.rot * sizeof(float), s>>>(a, d);
    } else {
        const int64_t pairs = a.tokens * (a.heads + 2 * hk) * (a.cache.dim / 2);
        auto fn = interleaved ? rope_append_kernel<T, C, true> : rope_append_kernel<T, C, false>;
        fn<<<(unsigned)std::min<int64_t>((pairs + 255) / 256, (int64_t)sms * 8), 256, 0, s>>>(a);
    }
    TMAC_CUDA_TRY(cudaGetLastError());
    return TMAC_OK;
}

}  // namespace
}  // namespace tmac

using namespace tmac;

extern "C" int tmac_rope_append(const tmac_paged_cache* cache, int type, const void* q, int64_t q_stride, const void* k,
                                int64_t k_stride, const void* v, int64_t v_stride, int heads, int tokens,
                                const float* bias, const int32_t* seq, const int32_t* pos, const int32_t* starts,
                                const int32_t* tables, int n_seq, int table_width, const float* cos,
                                const float* sin, int max_pos, int rot_dim, int interleaved, void* q_out, void* stream)
{
    RopeArgs a = {};
    int rc = check_cache(cache, &a.cache);
    if (rc) return rc;
    if (!type_bytes(type)) return fail(TMAC_ERR_TYPE, "type must be F32, F16 or BF16");
    if (tokens < 0 || heads <= 0 || heads > 65535) return fail(TMAC_ERR_SHAPE, "need heads > 0 and tokens >= 0");
    if (tokens == 0) return TMAC_OK;
    if (!q || !k || !v || !pos || !tables || !q_out) return fail(TMAC_ERR_INVALID, "NULL argument");
    if (n_seq <= 0 || table_width <= 0) return fail(TMAC_ERR_SHAPE, "need at least one table entry per sequence");
    if (!seq && n_seq < tokens) return fail(TMAC_ERR_SHAPE, "without seq there is one sequence per token");
    if (rot_dim < 0 || rot_dim % 2 || rot_dim > cache->head_dim)
        return fail(TMAC_ERR_SHAPE, "rot_dim must be even, 0 to head_dim");
    if (max_pos <= 0) return fail(TMAC_ERR_SHAPE, "max_pos must be positive");
    if (rot_dim && (!cos || !sin)) return fail(TMAC_ERR_INVALID, "NULL cos or sin");
    const int64_t d = cache->head_dim;
    if (q_stride < heads * d || k_stride < cache->kv_heads * d || v_stride < cache->kv_heads * d)
        return fail(TMAC_ERR_SHAPE, "token strides must cover a token's heads");
    const unsigned e = (unsigned)type_bytes(type);
    if ((uintptr_t)q % e || (uintptr_t)k % e || (uintptr_t)v % e || (uintptr_t)q_out % type_bytes(cache->type))
        return fail(TMAC_ERR_INVALID, "q, k, v and q_out must be aligned to their type");
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.q_out = q_out;
    a.bias = bias;
    a.seq = seq;
    a.pos = pos;
    a.starts = starts;
    a.tables = tables;
    a.cos = cos;
    a.sin = sin;
    a.tokens = tokens;
    a.heads = heads;
    a.n_seq = n_seq;
    a.table_width = table_width;
    a.max_pos = max_pos;
    a.rot = rot_dim;
    DeviceGuard dg(cache->device);
    if (!dg.ok) return fail(TMAC_ERR_NODEV, "no such CUDA device");
    if (!(a.err = device_error_word(cache->device))) return fail(TMAC_ERR_CUDA, "no device error word");
    const int sms = num_sms(cache->device);
    return with_type(type, [&](auto* t) {
        return with_type(cache->type, [&](auto* c) {
            return launch_rope<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(c)>>(
                a, interleaved != 0, sms, (cudaStream_t)stream);
        });
    });
}
