// rope_append.cu -- q, k and v of a step: bias, position rotation, and k and v
// stored into a paged cache (bias + apply_rope + cache writes of
// forward_layer_with_cache, sim/tmac_gguf.cpp:1528-1554, :1590-1622, for a batch of
// tokens of several sequences).
//
// For pair i of a head, with c = cos[pos][i], s = sin[pos][i]:
//   (a, z) -> (a c - z s, a s + z c),
// pairs (2i, 2i + 1) when interleaved, else (i, i + rot_dim / 2); the values past
// rot_dim pass through.  Products and sums are 32-bit, rounded once to the
// cache's type.
//
// Bound: HBM, every value is read once and written once.  Where the pointers,
// strides and head parts allow it a warp takes a token, its threads 8 adjoining
// values each (16 bytes of a 16-bit type), or 8 pairs of halves: a thread's place
// within the head stays the same from head to head, so its cosines and sines, and the
// token's page, are looked up once, while several heads' values are on their way.
// Other layouts take one pair per thread.
#include "serving.cuh"

#include <algorithm>

namespace tmac {
namespace {

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
                const float c = a.cos[(int64_t)p.pos * (a.rot / 2) + pair], s = a.sin[(int64_t)p.pos * (a.rot / 2) + pair];
                const float xr = __fadd_rn(__fmul_rn(x, c), -__fmul_rn(z, s));
                z = __fadd_rn(__fmul_rn(x, s), __fmul_rn(z, c));
                x = xr;
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
        const T* r = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = Elem<T>::load(r + i);
    }
};
template <typename T>
TMAC_DEV void store8(T* p, const float (&x)[8])
{
    Eight<T> e;
    T* r = reinterpret_cast<T*>(e.raw);
#pragma unroll
    for (int i = 0; i < 8; i++) Elem<T>::store(r + i, x[i]);
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

// Units of a q or k head: 8 values at a time (interleaved), or 8 pairs at a time of
// the rotated part and 8 values at a time of the rest; of a v head: 8 values at a time.
template <typename T, typename C, bool kInterleaved>
__global__ void __launch_bounds__(256) rope_append_vec_kernel(RopeArgs a)
{
    constexpr int kFlight = sizeof(T) == 4 ? 2 : 4;  // heads of a thread on their way
    const int d = a.cache.dim, hk = a.cache.kv_heads, lane = threadIdx.x & 31, shift = a.cache.page_shift;
    const int pairs8 = kInterleaved ? 0 : a.rot / 16, per_head = pairs8 + (kInterleaved ? d : d - a.rot) / 8;
    const int warps = (int)(gridDim.x * blockDim.x) >> 5;
    // heads of a pass, and this lane's head and unit within it
    const int at_once = 32 / per_head, my_row = lane / per_head, unit = lane - my_row * per_head;
    const bool halves = unit < pairs8;
    const int d0 = halves || kInterleaved ? unit * 8 : a.rot + (unit - pairs8) * 8, d1 = d0 + a.rot / 2;
    const bool turn = kInterleaved ? d0 < a.rot : halves;
    const int v_once = 32 / (d / 8), v_row = lane / (d / 8), v_d = lane % (d / 8) * 8;
    const int qk = a.heads + hk;
    for (int64_t t = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < a.tokens; t += warps) {
        const T *q = (const T*)a.q + t * a.q_stride, *k = (const T*)a.k + t * a.k_stride, *v = (const T*)a.v + t * a.v_stride;
        Place p;
        float c[8], s[8];
        for (int base = 0; base < qk; base += at_once * kFlight) {
            Eight<T> xr[kFlight], zr[kFlight];
#pragma unroll
            for (int f = 0; f < kFlight; f++) {
                const int row = base + f * at_once + my_row;
                if (my_row >= at_once || row >= qk) continue;
                const T* src = row < a.heads ? q + row * d : k + (row - a.heads) * d;
                xr[f].load(src + d0);
                if (halves) zr[f].load(src + d1);
            }
            if (base == 0) {
                p = place_of(a, t);
                if (turn && p.ok) {
                    const int64_t at = (int64_t)p.pos * (a.rot / 2);
                    if (kInterleaved) {
                        const float4 c4 = __ldg(reinterpret_cast<const float4*>(a.cos + at + d0 / 2));
                        const float4 s4 = __ldg(reinterpret_cast<const float4*>(a.sin + at + d0 / 2));
                        c[0] = c4.x, c[1] = c4.y, c[2] = c4.z, c[3] = c4.w;
                        s[0] = s4.x, s[1] = s4.y, s[2] = s4.z, s[3] = s4.w;
                    } else {
                        Eight<float> e;
                        e.load(a.cos + at + d0);
                        e.floats(c);
                        e.load(a.sin + at + d0);
                        e.floats(s);
                    }
                }
            }
            const int64_t page_row = p.page * hk;
#pragma unroll
            for (int f = 0; f < kFlight; f++) {
                const int row = base + f * at_once + my_row;
                if (my_row >= at_once || row >= qk) continue;
                const bool is_q = row < a.heads;
                C* dst;
                if (is_q)
                    dst = (C*)a.q_out + (t * a.heads + row) * d;
                else if (p.page >= 0)
                    dst = (C*)a.cache.k + (((page_row + row - a.heads) << shift) + p.slot) * d;
                else
                    continue;
                float x[8], z[8];
                xr[f].floats(x);
                if (halves) zr[f].floats(z);
                if (a.bias) {
                    add8(x, a.bias + row * d + d0);
                    if (halves) add8(z, a.bias + row * d + d1);
                }
                if (!p.ok) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = z[i] = 0.0f;
                } else if (turn) {
                    if (kInterleaved) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float y = __fadd_rn(__fmul_rn(x[2 * i], c[i]), -__fmul_rn(x[2 * i + 1], s[i]));
                            x[2 * i + 1] = __fadd_rn(__fmul_rn(x[2 * i], s[i]), __fmul_rn(x[2 * i + 1], c[i]));
                            x[2 * i] = y;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            const float y = __fadd_rn(__fmul_rn(x[i], c[i]), -__fmul_rn(z[i], s[i]));
                            z[i] = __fadd_rn(__fmul_rn(x[i], s[i]), __fmul_rn(z[i], c[i]));
                            x[i] = y;
                        }
                    }
                }
                store8(dst + d0, x);
                if (halves) store8(dst + d1, z);
            }
        }
        if (p.page < 0) continue;
        for (int base = 0; base < hk; base += v_once * kFlight) {
            Eight<T> xr[kFlight];
#pragma unroll
            for (int f = 0; f < kFlight; f++) {
                const int row = base + f * v_once + v_row;
                if (v_row < v_once && row < hk) xr[f].load(v + row * d + v_d);
            }
#pragma unroll
            for (int f = 0; f < kFlight; f++) {
                const int row = base + f * v_once + v_row;
                if (v_row >= v_once || row >= hk) continue;
                float x[8];
                xr[f].floats(x);
                if (a.bias) add8(x, a.bias + (qk + row) * d + v_d);
                store8((C*)a.cache.v + (((p.page * hk + row) << shift) + p.slot) * d + v_d, x);
            }
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
    const bool vec = vectors_fit<T, C>(a, interleaved);
    // a warp to a token, or a thread to a pair
    const int64_t threads = vec ? a.tokens * 32 : a.tokens * (a.heads + 2 * a.cache.kv_heads) * (a.cache.dim / 2);
    const int grid = (int)std::min<int64_t>((threads + 255) / 256, (int64_t)sms * 8);
    auto fn = vec ? interleaved ? rope_append_vec_kernel<T, C, true> : rope_append_vec_kernel<T, C, false>
                  : interleaved ? rope_append_kernel<T, C, true> : rope_append_kernel<T, C, false>;
    fn<<<grid, 256, 0, s>>>(a);
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
