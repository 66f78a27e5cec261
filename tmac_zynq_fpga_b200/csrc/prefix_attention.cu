// prefix_attention.cu -- attention of a batch whose sequences share a prefix,
// over a paged cache (the attention of forward_layer_with_cache,
// sim/tmac_gguf.cpp:1625-1660, for a batch of sequences and one or more query tokens
// of each).
//
// Query token i of sequence b sees the first prefix_lens[b] positions of the
// shared prefix and the first own_lens[b] - n_q + 1 + i of the sequence's own:
//   o = sum_j softmax_j(scale q.k_j) v_j   (0 when it sees none).
// The prefix's keys are read once for all sequences: its scores are one matrix
// product of all tokens' query rows, the own part one product per sequence.
// Both run as jobs of one grid, each a tile of rows (token, head of a key/value
// head's group) against a range of keys with a running maximum and sum; a job
// leaves (maximum, sum, unnormalised o), and attn_join_kernel joins a row's jobs.
#include "serving.cuh"

#include <algorithm>

namespace tmac {
namespace {

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
    // jobs: prefix tiles x key ranges x kv heads, then (sequence, tile) x key ranges x kv heads
    int p_tiles, p_splits, p_chunk;
    int o_tiles, o_splits, o_chunk;
    int64_t p_jobs;
    int parts;       // per row: p_splits + o_splits
    float* part_o;   // [tokens][heads][parts][dim]
    float2* part_ml; // [tokens][heads][parts]
    int* err;
};

TMAC_DEV int first_token(const AttnArgs& a, int b)
{
    const int t = a.q_start ? a.q_start[b] : b;
    return max(0, min(t, a.tokens));
}
// Query tokens of sequence b: at most max_q are computed, more is an error.
TMAC_DEV int token_count(const AttnArgs& a, int b)
{
    const int n = first_token(a, b + 1) - first_token(a, b);
    if (n > a.max_q) record_error(a.err, TMAC_ERR_BOUNDS);
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

// ---------------------------------------------------- 32-bit arithmetic ----
// Tiles of 8 rows per warp.  A warp takes 16 keys at a time: lane = (key, half
// of the rows) for the scores, lane = dims for the output.  With up to 8 rows
// in the job the four warps take different keys of a 64-key tile and join at
// the end; with more they take different rows and share the tile.
constexpr int kRows = 8, kTile = 64, kStep = 16, kSimtWarps = 4;

template <typename T, int D>
struct SimtSmem {
    float q[kSimtWarps * kRows][D];
    float p[kSimtWarps][kStep][kRows];
    float alpha[kSimtWarps][kRows];
    T k[kTile][D + 16 / sizeof(T)];
    T v[kTile][D];
    int limit[kSimtWarps * kRows], least_limit;
    int token[kSimtWarps * kRows], head[kSimtWarps * kRows];
};

// A job's rows and keys, the same for every kernel.
struct Job {
    int kvh, seq;             // seq < 0: prefix
    int row0, rows;           // of the sequence's (or all) tokens x group
    int key0, key1;           // key range
    int part;
    const int* pages;
    int token0;
};
template <int kJobRows>
TMAC_DEV bool find_job(const AttnArgs& a, Job* j)
{
    int64_t id = blockIdx.x;
    if (id < a.p_jobs) {
        const int tile = (int)(id % a.p_tiles);
        id /= a.p_tiles;
        j->kvh = (int)(id % a.cache.kv_heads);
        const int split = (int)(id / a.cache.kv_heads);
        j->seq = -1;
        j->row0 = tile * kJobRows;
        j->rows = min(kJobRows, a.tokens * a.group - j->row0);
        j->key0 = split * a.p_chunk;
        j->key1 = min(a.prefix_len, j->key0 + a.p_chunk);
        j->part = split;
        j->pages = a.prefix_pages;
        j->token0 = 0;
        return true;
    }
    id -= a.p_jobs;
    const int tile = (int)(id % a.o_tiles);
    id /= a.o_tiles;
    j->kvh = (int)(id % a.cache.kv_heads);
    id /= a.cache.kv_heads;
    const int split = (int)(id % a.o_splits);
    j->seq = (int)(id / a.o_splits);
    j->row0 = tile * kJobRows;
    j->rows = min(kJobRows, token_count(a, j->seq) * a.group - j->row0);
    j->key0 = split * a.o_chunk;
    j->key1 = min(own_len(a, j->seq), j->key0 + a.o_chunk);
    j->part = a.p_splits + split;
    j->pages = a.tables + (int64_t)j->seq * a.table_width;
    j->token0 = first_token(a, j->seq);
    return j->rows > 0 && j->key1 > j->key0;  // the join leaves other parts out
}
// The row's token and head, and how many keys of the job's kind it sees.
TMAC_DEV void find_row(const AttnArgs& a, const Job& j, int r, int* token, int* head, int* limit)
{
    const int row = j.row0 + r, i = row / a.group;
    *token = j.token0 + i;
    *head = j.kvh * a.group + row % a.group;
    *limit = j.seq < 0 ? prefix_seen(a, sequence_of(a, *token)) : own_len(a, j.seq) - token_count(a, j.seq) + 1 + i;
}
// First element of key `key`'s row in a pool; -1 for a page outside the pool
// (its rows count as zeros, and the error word says so).
TMAC_DEV int64_t key_row(const AttnArgs& a, const Job& j, int key)
{
    const int shift = a.cache.page_shift;
    const int64_t page = j.pages[key >> shift];
    if (page < 0 || page >= a.cache.n_pages) {
        record_error(a.err, TMAC_ERR_BOUNDS);
        return -1;
    }
    return (((page * a.cache.kv_heads + j.kvh) << shift) + (key & ((1 << shift) - 1))) * a.cache.dim;
}

template <typename T, int D>
__global__ void __launch_bounds__(kSimtWarps * 32) attn_simt_kernel(AttnArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    SimtSmem<T, D>& sh = *reinterpret_cast<SimtSmem<T, D>*>(smem);
    constexpr int kJobRows = kSimtWarps * kRows, kDims = D / 32, kVec = 16 / sizeof(T);
    Job j;
    if (!find_job<kJobRows>(a, &j)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool split_keys = j.rows <= kRows;
    if (threadIdx.x == 0) sh.least_limit = 0x7FFFFFFF;
    __syncthreads();
    for (int r = threadIdx.x; r < kJobRows; r += blockDim.x) {
        int token = 0, head = 0, limit = 0;
        if (r < j.rows) {
            find_row(a, j, r, &token, &head, &limit);
            atomicMin(&sh.least_limit, limit);
        }
        sh.token[r] = token;
        sh.head[r] = head;
        sh.limit[r] = limit;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kJobRows * D; i += blockDim.x) {
        const int r = i / D, d = i % D;
        sh.q[r][d] = r < j.rows ? __fmul_rn(a.scale, Elem<T>::load((const T*)a.q + sh.token[r] * a.q_stride + sh.head[r] * D + d))
                                : 0.0f;
    }

    const int r0 = split_keys ? 0 : warp * kRows;  // the warp's rows
    const int half = lane >> 4;                    // this lane's scores: rows half * 4 ..
    float m[4], l[4], o[kRows][kDims];
#pragma unroll
    for (int i = 0; i < 4; i++) m[i] = -INFINITY, l[i] = 0.0f;
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int c = 0; c < kDims; c++) o[r][c] = 0.0f;

    for (int tile = j.key0; tile < j.key1; tile += kTile) {
        __syncthreads();
        for (int i = threadIdx.x; i < kTile * (D / kVec); i += blockDim.x) {
            const int key = i / (D / kVec), c = i % (D / kVec) * kVec;
            uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
            if (tile + key < j.key1) {
                const int64_t at = key_row(a, j, tile + key);
                if (at >= 0) {
                    kx = *reinterpret_cast<const uint4*>((const T*)a.cache.k + at + c);
                    vx = *reinterpret_cast<const uint4*>((const T*)a.cache.v + at + c);
                }
            }
            *reinterpret_cast<uint4*>(&sh.k[key][c]) = kx;
            *reinterpret_cast<uint4*>(&sh.v[key][c]) = vx;
        }
        __syncthreads();
        for (int step = split_keys ? warp * kStep : 0; step < (split_keys ? (warp + 1) * kStep : kTile); step += kStep) {
            if (tile + step >= j.key1) break;
            const int kk = step + (lane & 15), key = tile + kk;
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int d = 0; d < D; d += kVec) {
                T kx[kVec];
                *reinterpret_cast<uint4*>(kx) = *reinterpret_cast<const uint4*>(&sh.k[kk][d]);
#pragma unroll
                for (int e = 0; e < kVec; e += 4) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 qv = *reinterpret_cast<const float4*>(&sh.q[r0 + half * 4 + i][d + e]);
                        s[i] = __fmaf_rn(qv.x, Elem<T>::load(kx + e), s[i]);
                        s[i] = __fmaf_rn(qv.y, Elem<T>::load(kx + e + 1), s[i]);
                        s[i] = __fmaf_rn(qv.z, Elem<T>::load(kx + e + 2), s[i]);
                        s[i] = __fmaf_rn(qv.w, Elem<T>::load(kx + e + 3), s[i]);
                    }
                }
            }
            float p[4], al[4];
            bool moved = false;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (key >= j.key1 || key >= sh.limit[r0 + half * 4 + i]) s[i] = -INFINITY;
                float mx = s[i];
#pragma unroll
                for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
                mx = fmaxf(mx, m[i]);
                al[i] = mx == m[i] ? 1.0f : expf(__fsub_rn(m[i], mx));
                moved |= mx != m[i];
                p[i] = s[i] == -INFINITY ? 0.0f : expf(__fsub_rn(s[i], mx));
                m[i] = mx;
                l[i] = __fmaf_rn(l[i], al[i], p[i]);
            }
            __syncwarp();
            *reinterpret_cast<float4*>(&sh.p[warp][lane & 15][half * 4]) = make_float4(p[0], p[1], p[2], p[3]);
            if (__any_sync(0xffffffffu, moved)) {
                if ((lane & 15) == 0)
                    *reinterpret_cast<float4*>(&sh.alpha[warp][half * 4]) = make_float4(al[0], al[1], al[2], al[3]);
                __syncwarp();
#pragma unroll
                for (int r = 0; r < kRows; r++)
#pragma unroll
                    for (int c = 0; c < kDims; c++) o[r][c] = __fmul_rn(o[r][c], sh.alpha[warp][r]);
            }
            __syncwarp();
            const bool some_masked = tile + step + kStep > sh.least_limit;
#pragma unroll 4
            for (int i = 0; i < kStep; i++) {
                float pr[kRows], vx[kDims];
#pragma unroll
                for (int r = 0; r < kRows; r++) pr[r] = sh.p[warp][i][r];
#pragma unroll
                for (int c = 0; c < kDims; c++) vx[c] = Elem<T>::load(&sh.v[step + i][lane * kDims + c]);
                // a row must not take 0 * inf from a key it does not see
#pragma unroll
                for (int r = 0; r < kRows; r++)
                    if (!some_masked || pr[r] != 0.0f)
#pragma unroll
                        for (int c = 0; c < kDims; c++) o[r][c] = __fmaf_rn(pr[r], vx[c], o[r][c]);
            }
        }
    }
    // row sums over the 16 key lanes
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) l[i] = __fadd_rn(l[i], __shfl_xor_sync(0xffffffffu, l[i], w));

    // the warps' results, joined over the warps when they split the keys
    __syncthreads();
    float* ml = reinterpret_cast<float*>(&sh.q[0][0]);        // [warps][8][2]
    float* ow = reinterpret_cast<float*>(&sh.k[0][0]);        // [warps][8][D]
    static_assert(sizeof(float) * kSimtWarps * kRows * D <= sizeof(sh.k) + sizeof(sh.v), "join space");
    if ((lane & 15) == 0)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            ml[(warp * kRows + half * 4 + i) * 2] = m[i];
            ml[(warp * kRows + half * 4 + i) * 2 + 1] = l[i];
        }
#pragma unroll
    for (int r = 0; r < kRows; r++)
#pragma unroll
        for (int c = 0; c < kDims; c++) ow[(warp * kRows + r) * D + lane * kDims + c] = o[r][c];
    __syncthreads();
    for (int i = threadIdx.x; i < j.rows * D; i += blockDim.x) {
        const int r = i / D, d = i % D;
        float mx, sum, val;
        if (split_keys) {
            mx = -INFINITY;
            for (int w = 0; w < kSimtWarps; w++) mx = fmaxf(mx, ml[(w * kRows + r) * 2]);
            sum = val = 0.0f;
            for (int w = 0; w < kSimtWarps; w++) {
                const float mw = ml[(w * kRows + r) * 2], lw = ml[(w * kRows + r) * 2 + 1];
                if (lw == 0.0f) continue;  // saw no key
                const float f = expf(__fsub_rn(mw, mx));
                sum = __fmaf_rn(f, lw, sum);
                val = __fmaf_rn(f, ow[(w * kRows + r) * D + d], val);
            }
        } else {
            mx = ml[r * 2];
            sum = ml[r * 2 + 1];
            val = ow[r * D + d];
        }
        const int64_t at = ((int64_t)sh.token[r] * a.heads + sh.head[r]) * a.parts + j.part;
        a.part_o[at * D + d] = val;
        if (d == 0) a.part_ml[at] = make_float2(mx, sum);
    }
}

// Joins the parts of one (token, head) per warp.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_join_kernel(AttnArgs a)
{
    constexpr int kDims = D / 32;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= (int64_t)a.tokens * a.heads) return;
    const int token = (int)(row / a.heads), head = (int)(row % a.heads), lane = threadIdx.x & 31;
    const int b = sequence_of(a, token);
    const int own = a.o_splits ? (own_len(a, b) + a.o_chunk - 1) / a.o_chunk : 0;
    const int n = a.p_splits + (token_count(a, b) > token - first_token(a, b) ? own : 0);
    const float2* ml = a.part_ml + row * a.parts;
    const float* po = a.part_o + row * a.parts * D + lane * kDims;
    float mx = -INFINITY;
    for (int s = lane; s < n; s += 32) mx = fmaxf(mx, ml[s].x);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
    float sum = 0.0f, o[kDims];
#pragma unroll
    for (int c = 0; c < kDims; c++) o[c] = 0.0f;
    for (int s = 0; s < n; s++) {
        const float2 p = ml[s];
        if (p.y == 0.0f) continue;  // saw no key
        const float f = expf(__fsub_rn(p.x, mx));
        sum = __fmaf_rn(f, p.y, sum);
#pragma unroll
        for (int c = 0; c < kDims; c++) o[c] = __fmaf_rn(f, po[(int64_t)s * D + c], o[c]);
    }
    T* out = (T*)a.out + token * a.out_stride + head * D + lane * kDims;
#pragma unroll
    for (int c = 0; c < kDims; c++) Elem<T>::store(out + c, sum == 0.0f ? 0.0f : __fdiv_rn(o[c], sum));
}

// How the work is cut: key ranges so that the grid has about two jobs per SM, of
// a tile at least.
int plan(AttnArgs* a, int sms)
{
    constexpr int kJobRows = kSimtWarps * kRows;
    const int hk = a->cache.kv_heads;
    auto ranges = [&](int64_t jobs, int keys, int* splits, int* chunk) {
        if (!jobs || !keys) {
            *splits = *chunk = 0;
            return;
        }
        const int tiles = (keys + kTile - 1) / kTile;
        const int64_t want = std::max<int64_t>(1, std::min<int64_t>(tiles, 2 * sms / jobs));
        *chunk = (int)((tiles + want - 1) / want) * kTile;
        *splits = (keys + *chunk - 1) / *chunk;
    };
    a->p_tiles = (int)(((int64_t)a->tokens * a->group + kJobRows - 1) / kJobRows);
    a->o_tiles = (int)(((int64_t)a->max_q * a->group + kJobRows - 1) / kJobRows);
    ranges((int64_t)a->p_tiles * hk, a->prefix_len, &a->p_splits, &a->p_chunk);
    ranges((int64_t)a->batch * a->o_tiles * hk, a->max_own, &a->o_splits, &a->o_chunk);
    a->p_jobs = (int64_t)a->p_tiles * hk * a->p_splits;
    a->parts = a->p_splits + a->o_splits;
    return TMAC_OK;
}

size_t workspace_bytes_of(const AttnArgs& a)
{
    const size_t rows = (size_t)a.tokens * a.heads * a.parts;
    return rows * (size_t)a.cache.dim * sizeof(float) + rows * sizeof(float2);
}

template <typename T, int D>
int launch_attention(const AttnArgs& a, cudaStream_t s)
{
    const int64_t jobs = a.p_jobs + (int64_t)a.batch * a.o_tiles * a.cache.kv_heads * a.o_splits;
    if (jobs > 0x7FFFFFFF) return fail(TMAC_ERR_SHAPE, "too many jobs for one grid");
    if (jobs) {
        auto fn = attn_simt_kernel<T, D>;
        TMAC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SimtSmem<T, D>)));
        fn<<<(unsigned)jobs, kSimtWarps * 32, sizeof(SimtSmem<T, D>), s>>>(a);
        TMAC_CUDA_TRY(cudaGetLastError());
    }
    attn_join_kernel<T, D><<<(unsigned)(((int64_t)a.tokens * a.heads + 3) / 4), 128, 0, s>>>(a);
    TMAC_CUDA_TRY(cudaGetLastError());
    return TMAC_OK;
}

// The checks and the plan both entries share.
int prepare(const tmac_paged_cache* cache, int heads, int tokens, int batch, int max_q, int prefix_len, int max_own,
            int table_width, AttnArgs* a)
{
    int rc = check_cache(cache, &a->cache);
    if (rc) return rc;
    if (cache->head_dim != 64 && cache->head_dim != 128) return fail(TMAC_ERR_SHAPE, "head_dim must be 64 or 128");
    if (heads <= 0 || heads % cache->kv_heads) return fail(TMAC_ERR_SHAPE, "heads must be a multiple of kv_heads");
    if (tokens < 0 || batch < 0 || max_q < 1) return fail(TMAC_ERR_SHAPE, "need tokens, batch >= 0 and max_q >= 1");
    if ((int64_t)tokens * heads > 0x7FFFFFFF || (int64_t)max_q * heads > 0x7FFFFFFF)
        return fail(TMAC_ERR_SHAPE, "too many query rows");
    if (prefix_len < 0 || max_own < 0 || prefix_len > 0x7FFFFF00 || max_own > 0x7FFFFF00)
        return fail(TMAC_ERR_SHAPE, "lengths out of range");
    if ((int64_t)table_width * cache->page_size < max_own) return fail(TMAC_ERR_SHAPE, "table_width does not cover max_own");
    a->heads = heads;
    a->group = heads / cache->kv_heads;
    a->tokens = tokens;
    a->batch = batch;
    a->max_q = max_q;
    a->prefix_len = prefix_len;
    a->max_own = max_own;
    a->table_width = table_width;
    if (tokens == 0) return TMAC_OK;
    return plan(a, num_sms(cache->device));
}

}  // namespace
}  // namespace tmac

using namespace tmac;

extern "C" int tmac_prefix_attention_workspace(const tmac_paged_cache* cache, int heads, int tokens, int batch,
                                               int max_q, int prefix_len, int max_own, size_t* bytes)
{
    if (!bytes) return fail(TMAC_ERR_INVALID, "NULL bytes");
    AttnArgs a = {};
    int rc = prepare(cache, heads, tokens, batch, max_q, prefix_len, max_own, 0x7FFFFFFF, &a);
    if (rc) return rc;
    *bytes = tokens ? workspace_bytes_of(a) : 0;
    return TMAC_OK;
}

extern "C" int tmac_prefix_attention(const tmac_paged_cache* cache, const void* q, int64_t q_stride, int heads,
                                     int tokens, int batch, const int32_t* q_start, int max_q,
                                     const int32_t* prefix_pages, int prefix_len, const int32_t* prefix_lens,
                                     const int32_t* tables, int table_width, const int32_t* own_lens, int max_own,
                                     float scale, void* out, int64_t out_stride, void* workspace,
                                     size_t workspace_bytes, void* stream)
{
    AttnArgs a = {};
    int rc = prepare(cache, heads, tokens, batch, max_q, prefix_len, max_own, table_width, &a);
    if (rc) return rc;
    if (tokens == 0) return TMAC_OK;
    if (!q || !out) return fail(TMAC_ERR_INVALID, "NULL argument");
    if (batch == 0) return fail(TMAC_ERR_SHAPE, "tokens without sequences");
    if (!q_start && (batch != tokens || max_q != 1))
        return fail(TMAC_ERR_SHAPE, "without q_start there is one token per sequence");
    if (prefix_len && !prefix_pages) return fail(TMAC_ERR_INVALID, "NULL prefix_pages");
    if (max_own && (!tables || !own_lens)) return fail(TMAC_ERR_INVALID, "NULL tables or own_lens");
    const int64_t row = (int64_t)heads * cache->head_dim;
    if (q_stride < row || out_stride < row) return fail(TMAC_ERR_SHAPE, "token strides must cover a token's heads");
    const unsigned e = (unsigned)type_bytes(cache->type);
    if ((uintptr_t)q % e || (uintptr_t)out % e) return fail(TMAC_ERR_INVALID, "q and out must be aligned to their type");
    const size_t need = workspace_bytes_of(a);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need))
        return fail(TMAC_ERR_INVALID, "workspace too small or not 16-byte aligned (tmac_prefix_attention_workspace)");
    a.q = q;
    a.q_stride = q_stride;
    a.out = out;
    a.out_stride = out_stride;
    a.q_start = q_start;
    a.prefix_pages = prefix_pages;
    a.prefix_lens = prefix_lens;
    a.tables = tables;
    a.own_lens = own_lens;
    a.scale = scale;
    a.part_o = (float*)workspace;
    a.part_ml = (float2*)(a.part_o + (size_t)tokens * heads * a.parts * cache->head_dim);
    DeviceGuard dg(cache->device);
    if (!dg.ok) return fail(TMAC_ERR_NODEV, "no such CUDA device");
    if (!(a.err = device_error_word(cache->device))) return fail(TMAC_ERR_CUDA, "no device error word");
    return with_type(cache->type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return cache->head_dim == 64 ? launch_attention<T, 64>(a, (cudaStream_t)stream)
                                     : launch_attention<T, 128>(a, (cudaStream_t)stream);
    });
}
