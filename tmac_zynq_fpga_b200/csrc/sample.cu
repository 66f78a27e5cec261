// sample.cu -- the next token of every sequence from its logits: temperature,
// top-k, top-p, min-p, and a draw from a given uniform number (sample_token,
// sim/tmac_gguf.cpp:1974-1990, keeps the top k and draws with rand()).
//
// For a row of logits l with inverse temperature t:
//   x = l t,   d = max x - x,   w = floor(2^32 exp(-d))
// x and d are 32-bit floats, w a whole number, so every sum of weights is exact
// and the same in any order: the drawn token does not depend on the grid or on
// the order of atomics.  A token of less than 2^-32 of the likeliest one's
// weight has weight 0 and is never drawn.  Tokens are ordered by (d, index).
// top-k keeps the first k, top-p the shortest first part whose weight reaches
// top_p times the weight of what top-k kept, min-p those with exp(-d) >= min_p;
// the token is the first kept index whose running weight passes u times the
// kept weight.
//
// One cluster of CTAs per row holds the row's d in shared memory, so the logits
// are read from HBM once.  The cut of top-k / top-p lies within a few units of
// the largest logit as a rule: one pass counts how many tokens lie within 1, 2, 4
// and 8 of it, and where at most kList of them hold the cut they are gathered in
// one CTA, sorted, and the draw ends there.  Otherwise (flat rows) the cut is
// found by radix selection on the bits of d over the whole cluster: a 1024-bin
// histogram of counts and weights per round, at most five rounds, each bin
// summed through distributed shared memory.
//
// Bound: HBM for large batches (every logit is read once), latency for one row.
#include "serving.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace tmac {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024;
constexpr float kBinScale = 45.5f;  // bins per unit of d in the first round; d < 22.2 where w > 0
constexpr int kMaxCluster = 16, kMaxSlice = 45000;
constexpr int kList = 2048, kWindows = 4;  // window i: d < 2^i
static_assert(kBins / kMaxCluster % 32 == 0, "a share's bins go to the lanes of a warp");
static_assert(kMaxSlice / kThreads < 255, "a thread's counts are bytes");

struct SampleArgs {
    const void* logits;
    int64_t stride;
    int vocab, slice;
    const float *u, *temperature;
    const int* top_k;
    const float *top_p, *min_p;
    int* tokens;
    float* probs;
};

struct Histogram {
    uint32_t cnt[kBins], hi[kBins], lo[kBins];  // this CTA's: counts, weights in two halves
    uint32_t mcnt[kBins];                       // this CTA's share of the bins, summed over the cluster
    unsigned long long mw[kBins];
};
struct List {
    unsigned long long key[kList], sorted[kList];  // bits(d) << 32 | index; by index, and in order
};
struct Shared {
    union {
        Histogram h;
        List list;
    };
    unsigned long long share_w, red_w[kWarps];
    uint32_t share_c, red_c[kWarps];
    float red_f[kWarps], cta_max;
    int cta_min_index;
    uint32_t warp_count[kWarps][kWindows], count[kWindows];  // tokens in each window: by warp, of the CTA
    uint32_t tie_count;
    unsigned long long kept;
    // broadcast of a search
    int found_bin, tie_index;
    uint32_t found_c, before_c;
    unsigned long long found_w, before_w;
    uint32_t n_keep;
};

TMAC_DEV float weight_exp(float d) { return expf(-d); }
TMAC_DEV unsigned long long weight_of(float e)
{
    return e >= 1.0f ? 0x100000000ull : (unsigned long long)(uint32_t)__fmul_rn(e, 4294967296.0f);
}
TMAC_DEV int first_bin(float d) { return min((int)__fmul_rn(d, kBinScale), kBins - 1); }

// The first part of a row's order that is kept: first_bin(d) < bin, or == bin and
// bits(d) <= key; among bits(d) == key only indexes up to tie_index.
struct Cut {
    int bin;
    uint32_t key;
    int tie_index;
    unsigned long long weight;  // of what it keeps
};
TMAC_DEV bool kept_by(const Cut& c, float d, int index)
{
    const int b = first_bin(d);
    if (b != c.bin) return b < c.bin;
    const uint32_t key = __float_as_uint(d);
    return key < c.key || (key == c.key && index <= c.tie_index);
}

template <typename V>
TMAC_DEV V warp_sum(V v)
{
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename V>
TMAC_DEV V warp_scan(V v)  // inclusive
{
    for (int o = 1; o < 32; o <<= 1) {
        const V up = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += up;
    }
    return v;
}

// floor(u * total), inside [0, total) whatever u is
TMAC_DEV unsigned long long pick_of(float u, unsigned long long total)
{
    const double at = __dmul_rn((double)u, (double)total);
    const unsigned long long pick = at > 0.0 ? (unsigned long long)at : 0;
    return pick < total ? pick : total - 1;
}

struct Row {
    cg::cluster_group cl;
    Shared* sh;
    float* d;        // this CTA's slice
    int n, begin;    // its length and first index
    int ranks, rank;

    // Calls f(value, local index) over the warp's own contiguous part, in order, 32 at a time.
    template <typename F>
    TMAC_DEV void walk(F&& f) const
    {
        const int per = (((n + kWarps - 1) / kWarps) + 31) & ~31;
        const int from = (threadIdx.x >> 5) * per, to = min(n, from + per);
        for (int i = from; i < to; i += 32) {
            const int j = i + (threadIdx.x & 31);
            f(j < to ? d[j] : INFINITY, j, j < to);
        }
    }

    // Adds the counts and weights of the local elements for which bin_of gives a bin.
    template <typename F>
    TMAC_DEV void histogram(F&& bin_of)
    {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh->h.cnt[i] = sh->h.hi[i] = sh->h.lo[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float v = d[i];
            const unsigned long long w = weight_of(weight_exp(v));
            if (!w) continue;
            const int b = bin_of(v);
            if (b < 0) continue;
            // a slice has at most kMaxSlice elements of at most 2^16 in either half: no overflow
            atomicAdd(&sh->h.cnt[b], 1u);
            atomicAdd(&sh->h.hi[b], (uint32_t)(w >> 16));
            atomicAdd(&sh->h.lo[b], (uint32_t)(w & 0xFFFF));
        }
        cl.sync();
        // this rank's share of the bins, over all ranks
        const int share = kBins / ranks;
        uint32_t c_sum = 0;
        unsigned long long w_sum = 0;
        for (int i = threadIdx.x; i < share; i += kThreads) {
            uint32_t c = 0;
            unsigned long long w = 0;
            for (int r = 0; r < ranks; r++) {
                const Shared* o = cl.map_shared_rank(sh, r);
                c += o->h.cnt[rank * share + i];
                w += ((unsigned long long)o->h.hi[rank * share + i] << 16) + o->h.lo[rank * share + i];
            }
            sh->h.mcnt[i] = c;
            sh->h.mw[i] = w;
            c_sum += c;
            w_sum += w;
        }
        c_sum = warp_sum(c_sum);
        w_sum = warp_sum(w_sum);
        if ((threadIdx.x & 31) == 0) {
            sh->red_c[threadIdx.x >> 5] = c_sum;
            sh->red_w[threadIdx.x >> 5] = w_sum;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < kWarps; i++) c_sum += sh->red_c[i], w_sum += sh->red_w[i];
            sh->share_c = c_sum;
            sh->share_w = w_sum;
        }
        cl.sync();
    }

    // The first bin at which the running count reaches k (k > 0) or the running
    // weight reaches t (k == 0), counting from base_c / base_w.  false: none does.
    // Warp 0 searches the ranks' shares, then the bins of the share that reaches it.
    TMAC_DEV bool search(uint32_t k, double t, uint32_t base_c, unsigned long long base_w)
    {
        if (threadIdx.x < 32) {
            const int lane = threadIdx.x, share = kBins / ranks;
            uint32_t c = 0;
            unsigned long long w = 0;
            if (lane < ranks) {
                const Shared* o = cl.map_shared_rank(sh, lane);
                c = o->share_c;
                w = o->share_w;
            }
            uint32_t up_c = base_c + warp_scan(c);
            unsigned long long up_w = base_w + warp_scan(w);
            const auto reached = [&](uint32_t n, unsigned long long m) { return k ? n >= k : (double)m >= t; };
            uint32_t hit = __ballot_sync(0xffffffffu, lane < ranks && reached(up_c, up_w));
            if (!hit) {
                if (lane == 0) sh->found_bin = -1;
            } else {
                const int r = __ffs(hit) - 1;
                base_c = __shfl_sync(0xffffffffu, up_c - c, r);
                base_w = __shfl_sync(0xffffffffu, up_w - w, r);
                const Shared* o = cl.map_shared_rank(sh, r);
                const int per = share / 32;  // adjoining bins of this lane
                c = 0;
                w = 0;
                for (int i = 0; i < per; i++) {
                    c += o->h.mcnt[lane * per + i];
                    w += o->h.mw[lane * per + i];
                }
                up_c = base_c + warp_scan(c);
                up_w = base_w + warp_scan(w);
                hit = __ballot_sync(0xffffffffu, reached(up_c, up_w));
                if (lane == __ffs(hit) - 1) {
                    c = up_c - c;
                    w = up_w - w;
                    for (int i = lane * per;; i++) {
                        const uint32_t bc = o->h.mcnt[i];
                        const unsigned long long bw = o->h.mw[i];
                        if (reached(c + bc, w + bw) || i + 1 == (lane + 1) * per) {
                            sh->found_bin = r * share + i;
                            sh->found_c = bc;
                            sh->found_w = bw;
                            sh->before_c = c;
                            sh->before_w = w;
                            break;
                        }
                        c += bc;
                        w += bw;
                    }
                }
            }
        }
        __syncthreads();
        return sh->found_bin >= 0;
    }

    // The index of the m-th element (from 1) with bits(d) == key, over the cluster.
    TMAC_DEV int tie(uint32_t key, uint32_t m)
    {
        uint32_t c = 0;
        walk([&](float v, int, bool in) { c += __popc(__ballot_sync(0xffffffffu, in && __float_as_uint(v) == key)); });
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) sh->red_c[warp] = c;
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t s = 0;
            for (int i = 0; i < kWarps; i++) s += sh->red_c[i];
            sh->tie_count = s;
        }
        cl.sync();
        uint32_t before = 0;
        for (int r = 0; r < rank; r++) before += cl.map_shared_rank(sh, r)->tie_count;
        for (int i = 0; i < warp; i++) before += sh->red_c[i];
        if (before < m && m <= before + c)
            walk([&](float v, int j, bool in) {
                const bool eq = in && __float_as_uint(v) == key;
                const uint32_t mask = __ballot_sync(0xffffffffu, eq);
                const uint32_t mine = before + __popc(mask & (0xFFFFFFFFu >> (31 - (threadIdx.x & 31))));
                if (eq && mine == m)
                    for (int r = 0; r < ranks; r++) cl.map_shared_rank(sh, r)->tie_index = begin + j;
                before += __popc(mask);
            });
        cl.sync();
        return sh->tie_index;
    }

    // Cuts the order after its first k elements (k > 0), or after the element at
    // which the running weight reaches t (k == 0).  Elements of weight 0 do not count.
    TMAC_DEV Cut select(uint32_t k, double t)
    {
        Cut cut = {kBins, 0xFFFFFFFFu, 0x7FFFFFFF, 0};
        histogram([&](float v) { return first_bin(v); });
        if (!search(k, t, 0, 0)) {  // fewer than k: all of them
            for (int r = 0; r < ranks; r++) cut.weight += cl.map_shared_rank(sh, r)->share_w;
            return cut;
        }
        cut.bin = sh->found_bin;
        // bits of d that the bin can hold, a little widened for the product's rounding
        uint32_t lo = __float_as_uint((float)cut.bin / kBinScale * 0.999999f);
        uint32_t span = __float_as_uint((float)(cut.bin + 1) / kBinScale * 1.000001f) - lo + 1;
        while (true) {
            const uint32_t found_c = sh->found_c, before_c = sh->before_c;
            const unsigned long long found_w = sh->found_w, before_w = sh->before_w;
            if (found_c == 1 || (k && before_c + found_c == k) || span == 1) {
                uint32_t m = found_c;
                unsigned long long w = found_w;
                if (span == 1) {
                    const unsigned long long each = found_w / found_c;
                    if (k)
                        m = k - before_c;
                    else  // the least m with before + m * each >= t
                        for (uint32_t a = 1, b = found_c; a <= b;) {
                            const uint32_t c = (a + b) / 2;
                            if ((double)(before_w + c * each) >= t) {
                                m = c;
                                b = c - 1;
                            } else {
                                a = c + 1;
                            }
                        }
                    w = m * each;
                }
                cut.weight = before_w + w;
                cut.key = cut.key == 0xFFFFFFFFu && span != 1 ? cut.key : lo + span - 1;
                if (m < found_c) cut.tie_index = tie(lo, m);
                return cut;
            }
            int shift = 0;
            while ((span - 1) >> shift >= kBins) shift++;
            cut.key = 0;  // from here on `lo + span` bounds the keys
            __syncthreads();  // every thread has read the last search
            histogram([&](float v) {
                const uint32_t o = __float_as_uint(v) - lo;
                return first_bin(v) == cut.bin && o < span ? (int)(o >> shift) : -1;
            });
            if (!search(k, t, before_c, before_w)) return cut;  // cannot happen: the bin holds the cut
            lo += (uint32_t)sh->found_bin << shift;
            span = 1u << shift;
        }
    }
};

// Exclusive running sum over the block of each thread's v; *total gets the sum of all.
TMAC_DEV unsigned long long block_scan(unsigned long long v, unsigned long long* red, unsigned long long* total)
{
    const unsigned long long up = warp_scan(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 31) red[threadIdx.x >> 5] = up;
    __syncthreads();
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWarps; i++) {
        const unsigned long long r = red[i];
        if (i < (int)(threadIdx.x >> 5)) before += r;
        all += r;
    }
    *total = all;
    return before + up - v;
}

// Sorts keys[0 .. n), n a power of two of 64 at least: a bitonic network, whose
// steps of distance 32 and less stay within the 64 keys of a warp.
TMAC_DEV void sort_keys(unsigned long long* keys, int n)
{
    for (int size = 2; size <= n; size <<= 1) {
        for (int step = size >> 1; step > 0; step >>= 1) {
            for (int t = threadIdx.x; t < n / 2; t += kThreads) {
                const int i = 2 * t - (t & (step - 1)), j = i + step;
                const unsigned long long x = keys[i], y = keys[j];
                if ((x > y) == ((i & size) == 0)) {
                    keys[i] = y;
                    keys[j] = x;
                }
            }
            if (step > 32 || (step == 1 && size >= 64))
                __syncthreads();
            else
                __syncwarp();
        }
    }
    __syncthreads();
}

// The cut and the draw over the n gathered tokens (in the order of their indexes).
// total: the row's weight when top_k is off.  false: top_p's cut lies beyond them.
TMAC_DEV bool draw_from_list(const SampleArgs& a, Shared* sh, int b, int n, int k, float p, float m, unsigned long long total)
{
    constexpr int kPer = kList / kThreads;
    List& list = sh->list;
    int size = 64;
    while (size < n) size <<= 1;
    for (int i = threadIdx.x; i < size; i += kThreads) list.sorted[i] = i < n ? list.key[i] : ~0ull;
    if (threadIdx.x == 0) sh->n_keep = 1;
    __syncthreads();
    sort_keys(list.sorted, size);
    const int n_k = k > 0 ? min(k, n) : n;

    float e[kPer];
    unsigned long long w[kPer], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int at = threadIdx.x * kPer + i;
        e[i] = at < n_k ? weight_exp(__uint_as_float((uint32_t)(list.sorted[at] >> 32))) : 0.0f;
        w[i] = at < n_k ? weight_of(e[i]) : 0;
        sum += w[i];
    }
    unsigned long long before = block_scan(sum, sh->red_w, &all);
    if (k > 0) total = all;
    const double t = __dmul_rn((double)p, (double)total);
    if (p < 1.0f && (double)all < t) return false;
    uint32_t keep = 0;  // the longest kept first part that ends with one of this thread's
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int at = threadIdx.x * kPer + i;
        if (at < n_k && (!(p < 1.0f) || (double)before < t) && e[i] >= m) keep = at + 1;
        before += w[i];
    }
    keep = __reduce_max_sync(0xffffffffu, keep);
    if ((threadIdx.x & 31) == 0 && keep) atomicMax(&sh->n_keep, keep);
    __syncthreads();
    const unsigned long long last = list.sorted[sh->n_keep - 1];

    sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int at = threadIdx.x * kPer + i;
        const unsigned long long key = at < n ? list.key[at] : ~0ull;
        w[i] = key <= last ? weight_of(weight_exp(__uint_as_float((uint32_t)(key >> 32)))) : 0;
        sum += w[i];
    }
    before = block_scan(sum, sh->red_w, &all);
    const unsigned long long pick = pick_of(a.u[b], all);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        if (w[i] && before <= pick && pick < before + w[i]) {
            a.tokens[b] = (int)(uint32_t)list.key[threadIdx.x * kPer + i];
            a.probs[b] = (float)__ddiv_rn((double)w[i], (double)all);
        }
        before += w[i];
    }
    return true;
}

// x = l * inv of the CTA's n logits into d, NaN as -inf; the largest of the thread's.
template <typename T>
TMAC_DEV float load_scaled(const T* l, int n, float inv, float* d)
{
    float mx = -INFINITY;
    auto put = [&](int i, float v) {
        float x = __fmul_rn(v, inv);
        if (isnan(x)) x = -INFINITY;
        d[i] = x;
        mx = fmaxf(mx, x);
    };
    constexpr int kVec = 16 / sizeof(T), kFlight = 4;
    const int head = min(n, (int)((16 - (uintptr_t)l % 16) % 16 / sizeof(T))), vecs = (n - head) / kVec;
    if ((int)threadIdx.x < head) put(threadIdx.x, Elem<T>::load(l + threadIdx.x));
    const int tail = head + vecs * kVec;
    if ((int)threadIdx.x < n - tail) put(tail + threadIdx.x, Elem<T>::load(l + tail + threadIdx.x));
    const uint4* v = reinterpret_cast<const uint4*>(l + head);
    for (int i0 = threadIdx.x; i0 < vecs; i0 += kThreads * kFlight) {
        uint4 r[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; f++)
            if (i0 + f * kThreads < vecs) r[f] = __ldg(v + i0 + f * kThreads);
#pragma unroll
        for (int f = 0; f < kFlight; f++) {
            if (i0 + f * kThreads >= vecs) break;
            T x[kVec];
            *reinterpret_cast<uint4*>(x) = r[f];
            float4 y[kVec / 4];
            float* yf = reinterpret_cast<float*>(y);
#pragma unroll
            for (int c = 0; c < kVec; c++) {
                yf[c] = __fmul_rn(Elem<T>::load(x + c), inv);
                if (isnan(yf[c])) yf[c] = -INFINITY;
                mx = fmaxf(mx, yf[c]);
            }
            // d is laid so that element `head` is 16-byte aligned
#pragma unroll
            for (int c = 0; c < kVec / 4; c++)
                *reinterpret_cast<float4*>(d + head + (i0 + f * kThreads) * kVec + 4 * c) = y[c];
        }
    }
    return mx;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    Row row = {cg::this_cluster()};
    row.sh = reinterpret_cast<Shared*>(smem);
    row.ranks = (int)row.cl.num_blocks();
    row.rank = (int)row.cl.block_rank();
    Shared* sh = row.sh;
    const int b = blockIdx.x / row.ranks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    row.begin = row.rank * a.slice;
    row.n = max(0, min(a.slice, a.vocab - row.begin));
    const T* l = (const T*)a.logits + b * a.stride + row.begin;
    // the first logit on a 16-byte boundary goes to one of shared memory
    const int head = (int)((16 - (uintptr_t)l % 16) % 16 / sizeof(T));
    row.d = reinterpret_cast<float*>(smem + (sizeof(Shared) + 15) / 16 * 16) + (4 - head % 4) % 4;

    const float temperature = a.temperature ? a.temperature[b] : 1.0f;
    float inv = __frcp_rn(temperature);
    const bool greedy = !(temperature > 0.0f) || isinf(inv);
    if (greedy) inv = 1.0f;
    int k = a.top_k ? a.top_k[b] : 0;
    if (k < 0 || k >= a.vocab) k = 0;
    float p = a.top_p ? a.top_p[b] : 1.0f;
    if (p <= 0.0f) {  // one token
        p = 1.0f;
        k = 1;
    }
    float m = a.min_p ? a.min_p[b] : 0.0f;
    m = m > 0.0f ? fminf(m, 1.0f) : 0.0f;

    // scaled logits, and the largest of the row
    float mx = load_scaled<T>(l, row.n, inv, row.d);
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) sh->red_f[warp] = mx;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWarps; i++) mx = fmaxf(mx, sh->red_f[i]);
        sh->cta_max = mx;
    }
    row.cl.sync();
    mx = lane < row.ranks ? row.cl.map_shared_rank(sh, lane)->cta_max : -INFINITY;
    for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = __shfl_sync(0xffffffffu, mx, 0);
    if (mx == -INFINITY) {  // nothing to choose from
        row.cl.sync();
        if (row.rank == 0 && threadIdx.x == 0) {
            a.tokens[b] = -1;
            a.probs[b] = 0.0f;
        }
        return;
    }

    if (greedy || k == 1) {  // the lowest index of the largest
        int first = 0x7FFFFFFF;
        for (int i = threadIdx.x; i < row.n; i += kThreads)
            if (row.d[i] == mx) first = min(first, row.begin + i);
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0) sh->red_c[warp] = (uint32_t)first;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < kWarps; i++) first = min(first, (int)sh->red_c[i]);
            sh->cta_min_index = first;
        }
        row.cl.sync();
        if (row.rank == 0 && threadIdx.x == 0) {
            for (int r = 1; r < row.ranks; r++) first = min(first, row.cl.map_shared_rank(sh, r)->cta_min_index);
            a.tokens[b] = first;
            a.probs[b] = 1.0f;
        }
        row.cl.sync();  // rank 0 has read the others' shared memory
        return;
    }

    // d, the tokens in each window, and the row's weight where the cut or the draw needs it
    const bool cuts = k > 0 || p < 1.0f, weigh = k <= 0;
    unsigned long long mine = 0;
    uint32_t counts = 0;  // of d < 1, [1, 2), [2, 4), [4, 8), a byte each
    row.walk([&](float x, int j, bool in) {
        if (!in) return;
        const float d = x == mx ? 0.0f : __fsub_rn(mx, x);
        row.d[j] = d;
        if (cuts && d < 8.0f) counts += 1u << (8 * max((int)(__float_as_uint(d) >> 23) - 126, 0));
        if (weigh) {
            const float e = weight_exp(d);
            // a cut by top-p is measured before min_p applies
            if (cuts || e >= m) mine += weight_of(e);
        }
    });
    mine = warp_sum(mine);
    if (lane == 0) sh->red_w[warp] = mine;
    if (cuts) {
        uint32_t c = 0;
#pragma unroll
        for (int i = 0; i < kWindows; i++) {
            c += (counts >> (8 * i)) & 0xFF;
            const uint32_t s = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0) sh->warp_count[warp][i] = s;
        }
    }
    __syncthreads();
    if (warp == 0) {
        unsigned long long s = lane < kWarps ? sh->red_w[lane] : 0;
        s = warp_sum(s);
        if (lane == 0) sh->kept = s;
        if (cuts)
#pragma unroll
            for (int i = 0; i < kWindows; i++) {
                const uint32_t c = __reduce_add_sync(0xffffffffu, lane < kWarps ? sh->warp_count[lane][i] : 0);
                if (lane == 0) sh->count[i] = c;
            }
    }
    row.cl.sync();
    unsigned long long total = 0, before = 0;
    for (int r = 0; r < row.ranks; r++) {
        const unsigned long long w = row.cl.map_shared_rank(sh, r)->kept;
        total += w;
        if (r < row.rank) before += w;
    }

    Cut cut = {kBins, 0xFFFFFFFFu, 0x7FFFFFFF, 0};
    if (cuts) {
        // the smallest window that holds top-k's cut, the largest that fits for top-p's alone
        int window = -1;
        uint32_t n = 0, offset = 0;
#pragma unroll
        for (int i = 0; i < kWindows; i++) {
            uint32_t c = lane < row.ranks ? row.cl.map_shared_rank(sh, lane)->count[i] : 0;
            const uint32_t up = warp_scan(c), all = __shfl_sync(0xffffffffu, up, 31);
            if (all <= kList && (k > 0 ? window < 0 && all >= (uint32_t)k : true)) {
                window = i;
                n = all;
                offset = __shfl_sync(0xffffffffu, up - c, row.rank);
            }
        }
        if (window >= 0) {
            for (int i = 0; i < warp; i++) offset += sh->warp_count[i][window];
            Shared* first = row.cl.map_shared_rank(sh, 0);
            const float limit = (float)(1 << window);
            row.walk([&](float d, int j, bool) {  // d past the slice is infinite
                const uint32_t hits = __ballot_sync(0xffffffffu, d < limit);
                if (d < limit)
                    first->list.key[offset + __popc(hits & ((1u << lane) - 1))] =
                        (unsigned long long)__float_as_uint(d) << 32 | (uint32_t)(row.begin + j);
                offset += __popc(hits);
            });
            row.cl.sync();
            bool done = true;
            if (row.rank == 0) done = draw_from_list(a, sh, b, (int)n, k, p, m, total);
            if (k > 0) return;  // the list holds the cut
            if (row.rank == 0 && threadIdx.x == 0) sh->n_keep = done;
            row.cl.sync();
            done = row.cl.map_shared_rank(sh, 0)->n_keep != 0;
            row.cl.sync();
            if (done) return;
        }
        if (k > 0) {
            cut = row.select((uint32_t)k, 0.0);
            total = cut.weight;
        }
        if (p < 1.0f) {
            __syncthreads();
            cut = row.select(0, __dmul_rn((double)p, (double)total));
        }
    }

    // the draw, in the order of the indexes
    auto kept_weight = [&](float v, int j, bool in) -> unsigned long long {
        if (!in || !kept_by(cut, v, row.begin + j)) return 0;
        const float e = weight_exp(v);
        return e >= m ? weight_of(e) : 0;
    };
    if (cuts) {
        mine = 0;
        row.walk([&](float v, int j, bool in) { mine += kept_weight(v, j, in); });
        mine = warp_sum(mine);
        __syncthreads();
        if (lane == 0) sh->red_w[warp] = mine;
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long s = 0;
            for (int i = 0; i < kWarps; i++) s += sh->red_w[i];
            sh->kept = s;
        }
        row.cl.sync();
        total = before = 0;
        for (int r = 0; r < row.ranks; r++) {
            const unsigned long long w = row.cl.map_shared_rank(sh, r)->kept;
            total += w;
            if (r < row.rank) before += w;
        }
    }
    for (int i = 0; i < warp; i++) before += sh->red_w[i];
    const unsigned long long pick = pick_of(a.u[b], total);
    if (before <= pick && pick < before + mine)
        row.walk([&](float v, int j, bool in) {
            const unsigned long long w = kept_weight(v, j, in), up_to = before + warp_scan(w);
            if (w && up_to > pick && up_to - w <= pick) {
                a.tokens[b] = row.begin + j;
                a.probs[b] = (float)__ddiv_rn((double)w, (double)total);
            }
            before = __shfl_sync(0xffffffffu, up_to, 31);
        });
    row.cl.sync();  // no CTA leaves while another reads its shared memory
}

template <typename T>
int launch_sample(const SampleArgs& a, int batch, int ranks, cudaStream_t s)
{
    const size_t smem = (sizeof(Shared) + 15) / 16 * 16 + ((size_t)a.slice + 3) * sizeof(float);
    auto fn = sample_kernel<T>;
    TMAC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    TMAC_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    TMAC_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, a));
    return TMAC_OK;
}

}  // namespace
}  // namespace tmac

using namespace tmac;

extern "C" int tmac_sample(const void* logits, int type, int64_t row_stride, int batch, int vocab, const float* u,
                           const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                           int32_t* tokens, float* probs, int device, void* stream)
{
    const int bytes = type_bytes(type);
    if (!bytes) return fail(TMAC_ERR_TYPE, "logits must be F32, F16 or BF16");
    if (batch < 0 || batch > 0x7FFFFFF) return fail(TMAC_ERR_SHAPE, "batch out of range");
    if (vocab <= 0 || vocab > kMaxCluster * kMaxSlice) return fail(TMAC_ERR_SHAPE, "vocab must be 1 to 720000");
    if (batch > 1 && row_stride < vocab) return fail(TMAC_ERR_SHAPE, "row_stride must cover a row");
    if (batch == 0) return TMAC_OK;
    if (!logits || !u || !tokens || !probs) return fail(TMAC_ERR_INVALID, "NULL argument");
    if ((uintptr_t)logits % bytes) return fail(TMAC_ERR_INVALID, "logits are not aligned to their type");
    SampleArgs a = {};
    a.logits = logits;
    a.stride = row_stride;
    a.vocab = vocab;
    a.u = u;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.tokens = tokens;
    a.probs = probs;
    const int ranks = vocab <= 4096 ? 1 : vocab <= 8 * kMaxSlice ? 8 : 16;
    a.slice = ((vocab + ranks - 1) / ranks + 7) & ~7;  // every rank's first logit is as aligned as the row's
    DeviceGuard dg(device);
    if (!dg.ok) return fail(TMAC_ERR_NODEV, "no such CUDA device");
    return with_type(type, [&](auto* t) {
        return launch_sample<std::remove_pointer_t<decltype(t)>>(a, batch, ranks, (cudaStream_t)stream);
    });
}
