// prefix_attention.cuh -- what the kernels of prefix_attention share: the arguments,
// how the grid's jobs, rows and key tiles are found, and where results go.
#pragma once

#include "serving.cuh"

#include <algorithm>
#include <type_traits>

namespace tmac {

struct AttnArgs {
    CacheDev cache;
    const void* q;
    int64_t q_stride;
    void* out;
    int64_t out_stride;
    int heads, group, tokens, batch, max_q;
    const int* q_start;
    const int *prefix_pages, *prefix_lens;
    int prefix_len;
    const int *tables, *own_lens;
    int table_width, max_own;
    float scale;
    // Jobs: prefix row tiles x kv heads x key ranges, then (sequence, row tile) x kv
    // heads x key ranges.  Key ranges are counted in tiles of kTile keys.
    bool alone;      // no prefix jobs: each sequence's keys are the prefix's and its own
    bool tc;         // the prefix jobs are the tcgen05 kernel's
    int p_tiles, p_splits, p_range;
    int o_tiles, o_splits, o_range;
    int64_t p_jobs;
    int parts;       // per row: p_splits + o_splits; 1: jobs write the result
    float* part_o;   // [tokens][heads][parts][dim]
    float2* part_ml; // [tokens][heads][parts]
    int* err;
    int device;
};

TMAC_DEV int first_token(const AttnArgs& a, int b)
{
    const int t = a.q_start ? a.q_start[b] : b;
    if (t < 0 || t > a.tokens) record_error(a.err, TMAC_ERR_BOUNDS);
    return max(0, min(t, a.tokens));
}
// Query tokens of sequence b: at most max_q are computed, more is an error.
TMAC_DEV int token_count(const AttnArgs& a, int b)
{
    const int n = first_token(a, b + 1) - first_token(a, b);
    if (n < 0 || n > a.max_q) record_error(a.err, TMAC_ERR_BOUNDS);
    return max(0, min(n, a.max_q));
}
TMAC_DEV int own_len(const AttnArgs& a, int b)
{
    const int n = a.own_lens[b];
    if (n > a.max_own) record_error(a.err, TMAC_ERR_BOUNDS);
    return max(0, min(n, a.max_own));
}
TMAC_DEV int prefix_seen(const AttnArgs& a, int b)
{
    if (!a.prefix_lens) return a.prefix_len;
    const int n = a.prefix_lens[b];
    if (n > a.prefix_len) record_error(a.err, TMAC_ERR_BOUNDS);
    return max(0, min(n, a.prefix_len));
}
TMAC_DEV int sequence_of(const AttnArgs& a, int token)
{
    if (!a.q_start) return token;
    int lo = 0, hi = a.batch - 1;  // the last sequence that starts at or before the token
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (a.q_start[mid] <= token)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}
// Whether a token's rows are computed, b its sequence_of: rows of tokens outside
// q_start[0] .. q_start[batch], and past a sequence's max_q, are zeros.
TMAC_DEV bool is_computed(const AttnArgs& a, int token, int b)
{
    const int i = token - first_token(a, b);
    return i >= 0 && i < token_count(a, b);
}

// Every sequence reads the prefix itself, in one job for all of its keys and without a
// join, up to so many key tiles in all (without a prefix up to kOwnTiles), and only where
// that is not more work than the join saves: the jobs are held by the GPU at once, or a
// sequence's query rows are at least kAloneRows for each tile of the prefix.  Against
// shared and joined jobs, us, tiles of prefix + own, query/key heads x dims, sequences;
// 16 bits:
//   3 + 1  14/2 x 64: 48 7.0 / 9.5, 384 17.0 / 22.8;  16/4 x 128: 48 10.8 / 12.8, 96 19.5 / 16.7
//   5 + 1  14/2 x 64: 48 8.6 / 9.9, 192 11.7 / 15.2;  8/8 x 64: 16 8.6 / 8.3, 192 37.4 / 22.3
//   7 + 1  14/2 x 64: 48 10.1 / 9.9;  32/8 x 128: 16 13.4 / 12.7, 192 80.4 / 49.3
//   0 + 8  14/2 x 64: 16 9.7 / 8.3, 192 13.1 / 19.4
// 32 bits:
//   1 + 1  14/2 x 64: 384 23.6 / 28.7;  16/4 x 128: 16 12.9 / 22.9, 192 66 / 55
//   3 + 1  14/2 x 64: 48 10.7 / 12.4, 384 36.8 / 33.1;  32/8 x 128: 192 201 / 119
constexpr int kAloneTiles16 = 6, kAloneTiles32 = 4, kOwnTiles16 = 8;
constexpr int kAloneRows16 = 2, kAloneRows32 = 5;
// The prefix goes to the tcgen05 kernel from so many rows on, and from so much work (rows
// x keys x kv heads).  There and in the mma kernel, us, with 64 own keys each, query/key
// heads, sequences x prefix:
//   64 dims   14/2  64 x 5000 (4.5 M) 18.3 / 15.7, 32 x 16384 (7.3 M) 20.2 / 20.0, 128 x 4096 (7.3 M) 20.2 / 22.3,
//             64 x 10000 (9.0 M) 20.2 / 21.4, 128 x 6000 (10.8 M) 21.6 / 26.1, 128 x 32768 (59 M) 41.9 / 78.8;
//             8/8  64 x 8192 (4.2 M) 22.9 / 20.3, 64 x 16384 (8.4 M) 25.5 / 25.0, 128 x 16384 (17 M) 31.5 / 37.5
//   128 dims  16/4  24 x 1100 (0.4 M) 14.9 / 13.5, 24 x 2500 (1.0 M) 15.9 / 15.0, 48 x 2200 (1.7 M) 16.0 / 20.6;
//             32/8  24 x 1300 (1.0 M) 15.1 / 16.6
constexpr int kTcRowsLeast = 48;
constexpr int64_t kTcWork64 = 8000000, kTcWork128 = 1000000;
constexpr int kTcRange = 4;  // tiles of its job at least: below, its start outweighs them
constexpr int kTile = 64, kWarps = 4, kThreads = kWarps * 32;

// A job's rows and keys, the same for every kernel.
struct Job {
    int kvh, seq;          // seq < 0: rows of all sequences, the prefix's keys
    int row0, rows, token0;
    int tile0, tile1;      // key tiles: first those of the prefix, then the own ones
    int p_tiles;           // of the prefix within them
    int p_keys, o_keys;    // keys in reach of the job
    int part;
};
TMAC_DEV int tiles_of(int keys) { return (keys + kTile - 1) / kTile; }
template <int kJobRows>
TMAC_DEV bool find_job(const AttnArgs& a, Job* j)
{
    uint32_t id = blockIdx.x;  // below 2^31; 32-bit divisions
    const uint32_t hk = (uint32_t)a.cache.kv_heads;
    if (id < (uint32_t)a.p_jobs) {
        const int tile = (int)(id % (uint32_t)a.p_tiles);
        id /= (uint32_t)a.p_tiles;
        j->kvh = (int)(id % hk);
        j->part = (int)(id / hk);
        j->seq = -1;
        j->token0 = 0;
        j->row0 = tile * kJobRows;
        j->rows = min(kJobRows, a.tokens * a.group - j->row0);
        j->p_keys = a.prefix_len;
        j->o_keys = 0;
        j->p_tiles = tiles_of(j->p_keys);
        j->tile0 = j->part * a.p_range;
        j->tile1 = min(j->p_tiles, j->tile0 + a.p_range);
        return true;
    }
    id -= (uint32_t)a.p_jobs;
    const int tile = (int)(id % (uint32_t)a.o_tiles);
    id /= (uint32_t)a.o_tiles;
    j->kvh = (int)(id % hk);
    id /= hk;
    const int split = (int)(id % (uint32_t)a.o_splits);
    j->seq = (int)(id / (uint32_t)a.o_splits);
    j->part = a.p_splits + split;
    j->token0 = first_token(a, j->seq);
    j->row0 = tile * kJobRows;
    j->rows = min(kJobRows, token_count(a, j->seq) * a.group - j->row0);
    j->p_keys = a.alone ? prefix_seen(a, j->seq) : 0;
    j->o_keys = a.max_own ? own_len(a, j->seq) : 0;
    j->p_tiles = tiles_of(j->p_keys);
    j->tile0 = split * a.o_range;
    j->tile1 = min(j->p_tiles + tiles_of(j->o_keys), j->tile0 + a.o_range);
    // without keys: the join leaves other parts out, but a lone part is the result
    return j->rows > 0 && (j->tile1 > j->tile0 || a.parts == 1);
}
// The row's token and head, and how many keys of the prefix and of its own it sees.
struct RowOf {
    int token, head, p_limit, o_limit;
};
TMAC_DEV RowOf find_row(const AttnArgs& a, const Job& j, int r)
{
    const int row = j.row0 + r, i = row / a.group;
    RowOf o;
    o.token = j.token0 + i;
    o.head = j.kvh * a.group + row % a.group;
    if (j.seq < 0) {
        o.p_limit = a.prefix_lens ? prefix_seen(a, sequence_of(a, o.token)) : a.prefix_len;
        o.o_limit = 0;
    } else {
        o.p_limit = j.p_keys;
        o.o_limit = max(0, j.o_keys - token_count(a, j.seq) + 1 + i);
    }
    return o;
}
// Where tile t's keys lie: the page list, the first key's number in it, the keys in reach.
struct TileOf {
    const int* pages;
    int key0, keys;
    bool prefix;
};
TMAC_DEV TileOf find_tile(const AttnArgs& a, const Job& j, int t)
{
    TileOf o;
    o.prefix = t < j.p_tiles;
    o.pages = o.prefix ? a.prefix_pages : a.tables + (int64_t)j.seq * a.table_width;
    o.key0 = (o.prefix ? t : t - j.p_tiles) * kTile;
    o.keys = o.prefix ? j.p_keys : j.o_keys;
    return o;
}
// kN adjoining values of a row's result from dim d on: the part's, or the rounded
// quotients when there is no other.
template <typename T, int D, int kN>
TMAC_DEV void put_results(const AttnArgs& a, const Job& j, const RowOf& row, int d, float m, float l, const float (&o)[kN])
{
    if (a.parts == 1) {
        T* to = (T*)a.out + row.token * a.out_stride + row.head * D + d;
        const float by = l == 0.0f ? 0.0f : __frcp_rn(l);
        float y[kN];
#pragma unroll
        for (int i = 0; i < kN; i++) y[i] = l == 0.0f ? 0.0f : sizeof(T) == 4 ? __fdiv_rn(o[i], l) : __fmul_rn(o[i], by);
        if constexpr (sizeof(T) == 2 && kN % 2 == 0) {
            if ((uintptr_t)to % 4 == 0) {
#pragma unroll
                for (int i = 0; i < kN / 2; i++) reinterpret_cast<uint32_t*>(to)[i] = pack2<T>(y[2 * i], y[2 * i + 1]);
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < kN; i++) Elem<T>::store(to + i, y[i]);
        return;
    }
    const int64_t at = ((int64_t)row.token * a.heads + row.head) * a.parts + j.part;
    float* to = a.part_o + at * D + d;
    if constexpr (kN == 4)
        *reinterpret_cast<float4*>(to) = make_float4(o[0], o[1], o[2], o[3]);
    else if constexpr (kN == 2)
        *reinterpret_cast<float2*>(to) = make_float2(o[0], o[1]);
    else
#pragma unroll
        for (int i = 0; i < kN; i++) to[i] = o[i];
    if (d == 0) a.part_ml[at] = make_float2(m, l);
}
// Maxima are in units of the exponential's base: e in 32 bits, where the difference
// of two scores is formed before it is scaled; 2 in 16 bits, one multiplication less.
TMAC_DEV float exp2_fast(float x)  // within 2^-22 relatively, tiny ones as 0
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <typename T>
TMAC_DEV float power(float x)
{
    return sizeof(T) == 4 ? expf(x) : exp2_fast(x);
}

// Row r of a job by one warp, key by key on the FMA units and only over the keys that it
// sees: for rows whose products met something that is not finite.  The matrix products
// add 0 * v for a key that a row does not see, which an infinite or NaN v turns into
// NaN; a large 32-bit number has no split; and weights above 1 overflow with large v
// before the division by their sum.
template <typename T, int D>
__device__ __noinline__ void row_by_keys(const AttnArgs& a, Job j, int r)
{
    constexpr int kPer = D / 32;  // adjoining dims of a lane
    const int d = (threadIdx.x & 31) * kPer, shift = a.cache.page_shift;
    const RowOf row = find_row(a, j, r);
    const float scale = sizeof(T) == 4 ? a.scale : __fmul_rn(a.scale, 1.44269504f);  // as power's base
    float q[kPer], o[kPer], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        q[i] = Elem<T>::load((const T*)a.q + row.token * a.q_stride + row.head * D + d + i);
        o[i] = 0.0f;
    }
    for (int t = j.tile0; t < j.tile1; t++) {
        const TileOf tile = find_tile(a, j, t);
        const int end = min(min(tile.prefix ? row.p_limit : row.o_limit, tile.keys), tile.key0 + kTile);
        for (int key = tile.key0; key < end; key++) {
            const int64_t page = __ldg(tile.pages + (key >> shift));
            const bool known = page >= 0 && page < a.cache.n_pages;  // else zeros; recorded before
            const int64_t at = known ? (((page * a.cache.kv_heads + j.kvh) << shift) + (key & ((1 << shift) - 1))) * D + d : 0;
            float s = 0.0f, v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                s = __fmaf_rn(q[i], known ? Elem<T>::load((const T*)a.cache.k + at + i) : 0.0f, s);
                v[i] = known ? Elem<T>::load((const T*)a.cache.v + at + i) : 0.0f;
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, w));
            s = __fmul_rn(s, scale);
            const float mx = fmaxf(m, s), al = m == mx ? 1.0f : power<T>(__fsub_rn(m, mx));
            const float p = s == -INFINITY ? 0.0f : power<T>(__fsub_rn(s, mx));
            l = __fmaf_rn(l, al, p);
#pragma unroll
            for (int i = 0; i < kPer; i++) {
                o[i] = __fmul_rn(o[i], al);
                if (p != 0.0f) o[i] = __fmaf_rn(p, v[i], o[i]);
            }
            m = mx;
        }
    }
    put_results<T, D, kPer>(a, j, row, d, m, l, o);
}

// Zeros for the rows that belong to no sequence or lie past its max_q, where jobs write
// the result and no join follows: by jobs of the prefix for their own rows, when all
// threads have written theirs; by a sequence's first job up to the next sequence.
template <typename T, int D, int kJobRows>
__device__ __noinline__ void clear_rows(const AttnArgs& a)
{
    Job j;
    find_job<kJobRows>(a, &j);
    const int width = a.group * D;
    const auto clear = [&](int from, int to) {
        for (int64_t i = threadIdx.x; i < (int64_t)(to - from) * width; i += blockDim.x)
            Elem<T>::store((T*)a.out + (from + i / width) * a.out_stride + j.kvh * width + i % width, 0.0f);
    };
    if (j.seq < 0) {
        __syncthreads();
        for (int token = j.row0 / a.group; token * a.group < j.row0 + j.rows; token++)
            if (!is_computed(a, token, sequence_of(a, token))) {
                const int first = max(0, j.row0 - token * a.group), last = min(a.group, j.row0 + j.rows - token * a.group);
                for (int i = first * D + threadIdx.x; i < last * D; i += blockDim.x)
                    Elem<T>::store((T*)a.out + token * a.out_stride + j.kvh * width + i, 0.0f);
            }
    } else if (j.row0 == 0) {
        if (j.seq == 0) clear(0, first_token(a, 0));
        clear(j.token0 + token_count(a, j.seq), j.seq + 1 < a.batch ? first_token(a, j.seq + 1) : a.tokens);
    }
}

// prefix_attention_tc.cu: the prefix's jobs of 16-bit elements on tcgen05.
constexpr int kTcRows = 128;  // rows of a job
int launch_prefix_tc(const AttnArgs& a, int type, cudaStream_t s);

}  // namespace tmac
