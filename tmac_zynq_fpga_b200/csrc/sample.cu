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
// A row belongs to one cluster of CTAs.  With few rows up to eight CTAs hold its x in
// shared memory, so the logits are read once.  With many rows (more than the SMs
// hold that way) as few CTAs read the logits again for each pass, mostly from L2:
// then every row is in flight at once, instead of waiting for others' clusters.
// Three ways to the cut:
//  * top-k: the k-th largest of the threads' own maxima bounds the k-th largest
//    logit from below, and closely, since a thread holds a few dozen logits.  The
//    tokens above the bound are gathered in one CTA, sorted, and the draw ends there.
//    Rows that are not held list the tokens in the pass that finds the maxima, above a
//    bound from the row's first quarter, and read the logits again only where that
//    bound proves too high (k up to 200 of 256 x 151936: 54 us, 74 with the second pass).
//  * top-p alone: its cut may lie anywhere, so a histogram of the weights over d
//    (bins of 1/22) is summed through distributed shared memory; every CTA then
//    gathers and sorts the tokens of the one bin that holds the cut.
//  * where the tokens to gather do not fit (many equal ones, a large k): radix
//    selection on the bits of d, one histogram per round, at most five rounds.
//
// Bound: HBM and a row's sort for large batches (top-k of 256 rows of 151936 32-bit
// logits 40 us at k = 40, 3900 GB/s; 54 at k up to 199 with top-p), the exchanges of a
// cluster for one row (top-k 9.8 us, top-p 27).  Of the latter's 46000 clocks the
// histogram takes 8500, merging and searching it 7000, listing and ordering the
// cut's bin 14000, the draw 11000.
#include "serving.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace tmac {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 512;
constexpr float kBinScale = 22.5f;  // bins per unit of d in the first round; d < 22.2 where w > 0
constexpr int kCluster = 8, kMaxCluster = 16, kMaxSlice = 45000, kMaxVocab = kMaxCluster * kMaxSlice;
constexpr int kList = 2048;                                    // tokens gathered in one CTA
constexpr int kFew = 256;                                      // of these, so many are ordered by counting
static_assert(kThreads >= kBins && kThreads * kMaxCluster / kBins <= 32, "the threads of a bin are lanes of a warp");
static_assert(kBins / kMaxCluster % 32 == 0, "a share's bins go to the lanes of a warp");
// Resident rows list up to 512 tokens per CTA and keep their x; others have the room for more.
template <bool kResident>
struct Layout {
    static constexpr int kLocal = kResident ? 512 : kList;
    // Steps of the bounds on d, from 1/16 to 16: 8 or 16 to an octave.  The finer ones
    // list fewer tokens, but eight CTAs read each other's counts: 9.8 and 11.6 us a row.
    static constexpr int kStepShift = kResident ? 20 : 19, kSteps = kResident ? 64 : 128, kFirstStep = (127 - 4) << (23 - kStepShift);
    static constexpr int kChunkVecs = kResident ? 64 : 256;  // float4 of a chunk of the draw
    static constexpr int kChunks = ((kResident ? kMaxSlice : kMaxVocab) + 6) / (4 * kChunkVecs) + 1;
};

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

struct Shared {
    union {
        struct {
            uint32_t cnt[kBins], hi[kBins], lo[kBins];  // this CTA's histogram: counts, weights in two words
        };
        alignas(16) unsigned long long pairs[2 * kFew];  // of count_before, when the histogram has been searched
    };
    uint32_t mcnt[kBins];                       // this CTA's share of the bins, summed over the cluster
    unsigned long long mw[kBins];
    unsigned long long key[kList];  // gathered tokens: bits(d) << 32 | index
    uint32_t n_few;
    unsigned long long share_w, red_w[kWarps];
    uint32_t share_c, red_c[kWarps];
    float red_f[kWarps], cta_max, least;  // least: every token of this CTA whose x is no less is listed
    int cta_min_index;
    alignas(16) uint32_t maxima[Layout<false>::kSteps];  // the threads' maxima by their distance from the row's
    uint32_t n_local;                    // listed tokens; more than kLocal: not all of them
    uint32_t n_keep;
    unsigned long long kept, cut_weight, cut_key;
    int chunk;  // the draw's
    unsigned long long chunk_before;
    // broadcast of a search
    int found_bin, tie_index;
    uint32_t found_c, before_c;
    unsigned long long found_w, before_w;
};

constexpr size_t kSharedBytes = (sizeof(Shared) + 15) / 16 * 16;
template <bool kResident>
constexpr size_t list_bytes()  // up to where x starts
{
    return (kSharedBytes + sizeof(unsigned long long) * (Layout<kResident>::kLocal + Layout<kResident>::kChunks) + 15) / 16 * 16;
}

template <bool kResident>
size_t sample_bytes(int slice)
{
    return list_bytes<kResident>() + (kResident ? ((size_t)slice + 6) * sizeof(float) : 0);
}

TMAC_DEV float weight_exp(float d) { return expf(-d); }
TMAC_DEV unsigned long long weight_of(float e)
{
    // the conversion saturates at 2^32 - 1, which e = 1 alone reaches
    return (unsigned long long)(uint32_t)__float2uint_rz(__fmul_rn(e, 4294967296.0f)) + (e >= 1.0f);
}
// Tokens of weight 0 lie past the last bin: they are asked for only where it does not matter.
TMAC_DEV int first_bin(float d) { return __float2int_rz(__fmul_rn(d, kBinScale)); }

TMAC_DEV unsigned long long order_key(float d, int index)
{
    return (unsigned long long)__float_as_uint(d) << 32 | (uint32_t)index;
}
// The first part of a row's order that is kept, up to the key `last`, which lies in `bin`.
struct Cut {
    int bin = kBins;
    float from = INFINITY, to = INFINITY;  // bounds on the d of the bin, widened for the product's rounding
    unsigned long long last = ~0ull;
    unsigned long long weight = 0;  // of what it keeps
    TMAC_DEV void set_bin(int b)
    {
        bin = b;
        from = __fmul_rn(__fdiv_rn((float)b, kBinScale), 0.999999f);
        to = __fmul_rn(__fdiv_rn((float)(b + 1), kBinScale), 1.000001f);
    }
};
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

// Sorts keys[0 .. n), n up to kList, which must have room for the next power of two
// (64 at least): a bitonic network, whose steps of distance 32 and less stay
// within the 64 keys of a warp.
TMAC_DEV void sort_keys(unsigned long long* keys, int count)
{
    int n = 64;
    while (n < count) n <<= 1;
    for (int i = count + threadIdx.x; i < n; i += kThreads) keys[i] = ~0ull;
    __syncthreads();
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

// floor(u * total), inside [0, total) whatever u is
TMAC_DEV unsigned long long pick_of(float u, unsigned long long total)
{
    const double at = __dmul_rn((double)u, (double)total);
    const unsigned long long pick = at > 0.0 ? (unsigned long long)at : 0;
    return pick < total ? pick : total - 1;
}

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

// Running sums in the order of few keys, by counting: threads 0 .. n - 1 hold a key
// and a weight each; *rank and *before get the number of smaller keys and their weight.
// `pairs` has room for 2 n numbers.
TMAC_DEV void count_before(unsigned long long* pairs, int n, unsigned long long key, unsigned long long w, int* rank,
                           unsigned long long* before)
{
    __syncthreads();
    if ((int)threadIdx.x < n) {
        pairs[2 * threadIdx.x] = key;
        pairs[2 * threadIdx.x + 1] = w;
    }
    __syncthreads();
    int r = 0;
    unsigned long long b = 0;
    if ((int)threadIdx.x < n) {
        const ulonglong2* p = reinterpret_cast<const ulonglong2*>(pairs);
#pragma unroll 4
        for (int k = 0; k < n; k++) {
            const ulonglong2 o = p[k];
            const bool less = o.x < key;
            r += less;
            b += less ? o.y : 0;
        }
    }
    *rank = r;
    *before = b;
}
// The sum over the first n threads' v, n up to kFew, to all.
TMAC_DEV unsigned long long sum_few(unsigned long long v, int n, unsigned long long* red)
{
    __syncthreads();
    if ((int)(threadIdx.x & ~31u) < n) {
        v = warp_sum((int)threadIdx.x < n ? v : 0);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    }
    __syncthreads();
    unsigned long long s = 0;
    for (int i = 0; i < (n + 31) / 32; i++) s += red[i];
    return s;
}

template <typename T, bool kResident>
struct Row {
    using L = Layout<kResident>;
    cg::cluster_group cl;
    Shared* sh;
    unsigned long long *local, *chunks;  // listed tokens; the draw's sums
    float* x;                            // resident: this CTA's scaled logits
    const T* l;                          // its logits
    float inv;
    int n, begin;  // their number and first index
    int pad;       // so many before the first make whole vectors of 4; -inf there and behind
    int ranks, rank;
    float mx;      // the row's largest
    bool infinite; // it is infinite: those share the weight, at d = 0

    TMAC_DEV float scaled(T v) const { return fmaxf(__fmul_rn(Elem<T>::load(&v), inv), -INFINITY); }  // NaN: -inf
    TMAC_DEV int vectors() const { return (pad + n + 3) / 4; }
    // Vector i holds the local indexes from 4 i - pad on.  As it lies in memory, for
    // one that is whole within the slice:
    using Raw = std::conditional_t<kResident || sizeof(T) == 4, uint4, uint2>;
    TMAC_DEV Raw raw4(int i) const
    {
        if constexpr (kResident)
            return reinterpret_cast<const uint4*>(x - pad)[i];
        else
            return __ldg(reinterpret_cast<const Raw*>(l + 4 * i - pad));
    }
    TMAC_DEV float4 from_raw(const Raw& raw) const
    {
        if constexpr (kResident) {
            return *reinterpret_cast<const float4*>(&raw);
        } else {
            const T* r = reinterpret_cast<const T*>(&raw);
            return make_float4(scaled(r[0]), scaled(r[1]), scaled(r[2]), scaled(r[3]));
        }
    }
    TMAC_DEV float4 load4(int i) const
    {
        const int j = 4 * i - pad;
        if constexpr (!kResident) {
            if (j < 0 || j + 4 > n) {
                float e[4];
#pragma unroll
                for (int c = 0; c < 4; c++) e[c] = j + c >= 0 && j + c < n ? scaled(l[j + c]) : -INFINITY;
                return make_float4(e[0], e[1], e[2], e[3]);
            }
        }
        return from_raw(raw4(i));
    }
    TMAC_DEV float d_of(float v) const
    {
        if (infinite) return v == INFINITY ? 0.0f : INFINITY;
        return __fsub_rn(mx, v);
    }
    // Calls f(d of four, local index of the first) for every `stride`-th vector from
    // `from` to `to`; indexes outside the slice have d = inf.
    template <typename F>
    TMAC_DEV void vectors(int from, int to, int stride, F&& f) const
    {
        constexpr int kFlight = 4;  // 2 costs 5-10% where rows are read anew, 8 the same in 16 bits
        const auto use = [&](const float4& q, int i) {
            const float e[4] = {d_of(q.x), d_of(q.y), d_of(q.z), d_of(q.w)};
            f(e, 4 * i - pad);
        };
        int i = from;
        if (!kResident && 4 * i < pad && i < to) {  // starts before the slice
            use(load4(i), i);
            i += stride;
        }
        const int whole = kResident ? to : min(to, (pad + n) / 4);
        for (; i + (kFlight - 1) * stride < whole; i += kFlight * stride) {  // several loads in flight
            Raw raw[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; u++) raw[u] = raw4(i + u * stride);
#pragma unroll
            for (int u = 0; u < kFlight; u++) use(from_raw(raw[u]), i + u * stride);
        }
        for (; i < to; i += stride) use(load4(i), i);
    }

    // Lists those of a vector's four tokens that `wanted` marks, with these d (or x).
    TMAC_DEV void put(const float (&v)[4], const bool (&wanted)[4], int index)
    {
        const volatile uint32_t* listed = &sh->n_local;
        const uint32_t count = (uint32_t)wanted[0] + wanted[1] + wanted[2] + wanted[3];
        if (!count || *listed > L::kLocal) return;
        uint32_t at = atomicAdd(&sh->n_local, count);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (wanted[c] && at < L::kLocal) local[at] = order_key(v[c], index + c);
            at += wanted[c];
        }
    }
    // Lists the tokens with from <= d < to for which `which` holds too, as long as
    // they fit, in any order, and waits for the cluster's lists.
    template <typename F>
    TMAC_DEV void list(float from, float to, F&& which)
    {
        if (threadIdx.x == 0) sh->n_local = 0;
        __syncthreads();
        vectors(threadIdx.x, vectors(), kThreads, [&](const float (&e)[4], int j) {
            bool wanted[4];
#pragma unroll
            for (int c = 0; c < 4; c++) wanted[c] = e[c] < to && e[c] >= from && which(e[c]);
            put(e, wanted, begin + j);
        });
        cl.sync();
    }

    // The bound below which, by `maxima`, k of the threads have their maximum's distance, or inf.
    // Steps of a lane, and what counts_of gives: their counts.
    static constexpr int kMine = L::kSteps / 32;
    using Counts = std::conditional_t<kMine == 4, uint4, uint2>;
    template <typename F>
    static TMAC_DEV float bound_of(uint32_t k, F&& counts_of)
    {
        const Counts c = counts_of();
        uint32_t n[kMine], all = 0;
#pragma unroll
        for (int i = 0; i < kMine; i++) n[i] = all += reinterpret_cast<const uint32_t*>(&c)[i];
        const uint32_t up = warp_scan(all), hit = __ballot_sync(0xffffffffu, up >= k);
        if (!hit) return INFINITY;
        int less = 0;
#pragma unroll
        for (int i = 0; i < kMine - 1; i++) less += up - all + n[i] < k;
        const int at = __ffs(hit) - 1, step = kMine * at + __shfl_sync(0xffffffffu, less, at);
        return __uint_as_float((uint32_t)(L::kFirstStep + step + 1) << L::kStepShift);
    }
    TMAC_DEV void count_maximum(float d)
    {
        const int step = (int)(__float_as_uint(d) >> L::kStepShift) - L::kFirstStep;
        if (step < L::kSteps) atomicAdd(&sh->maxima[max(step, 0)], 1u);
    }
    // One pass over the logits for the largest x, in which the tokens are listed, as x and
    // index, that are likely to be the first k and some more: those from `least` on, the
    // least of the threads' (k / 2 + 16) largest maxima over the slice's first quarter,
    // where k / 4 of them are to be expected.  The caller sees afterwards whether they
    // are enough.  mx is 0 meanwhile: d is -x.
    TMAC_DEV float max_and_list(uint32_t k, float* least)
    {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = vectors() / 4;
        float own = -INFINITY;
        vectors(threadIdx.x, part, kThreads, [&](const float (&e)[4], int) {
            own = fmaxf(own, -fminf(fminf(e[0], e[1]), fminf(e[2], e[3])));
        });
        float top = own;
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) sh->red_f[warp] = top;
        if (threadIdx.x < L::kSteps) sh->maxima[threadIdx.x] = 0;
        if (threadIdx.x == 0) sh->n_local = 0;
        __syncthreads();
        top = lane < kWarps ? sh->red_f[lane] : -INFINITY;
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const bool finite = fabsf(top) < INFINITY;
        if (finite) count_maximum(__fsub_rn(top, own));
        __syncthreads();
        const float d = bound_of(min(k, k / 2 + 16), [&] { return reinterpret_cast<const Counts*>(sh->maxima)[lane]; });
        // a little less, so that the distances of the k from the row's largest stay below it
        const float from = __fsub_rn(__fsub_rn(top, d), __fmul_rn(1e-6f, fmaxf(fabsf(top), d)));
        *least = finite && d < INFINITY ? from : INFINITY;
        const float to = -*least;
        const auto take = [&](const float (&e)[4], int j) {
            float v[4];
            bool wanted[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                v[c] = -e[c];
                own = fmaxf(own, v[c]);
                wanted[c] = e[c] <= to;
            }
            put(v, wanted, begin + j);
        };
        vectors(threadIdx.x, part, kThreads, take);
        vectors(part + threadIdx.x, vectors(), kThreads, take);
        return own;
    }
    // Of the tokens that max_and_list listed, those with d < to, listed as list() does.
    TMAC_DEV void relist(float to)
    {
        constexpr int kPer = (L::kLocal + kThreads - 1) / kThreads;
        const int n = (int)sh->n_local;
        unsigned long long key[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = threadIdx.x + i * kThreads;
            key[i] = ~0ull;
            if (at >= n) continue;
            const float d = d_of(__uint_as_float((uint32_t)(local[at] >> 32)));
            if (d < to) key[i] = order_key(d, (int)(uint32_t)local[at]);
        }
        __syncthreads();
        if (threadIdx.x == 0) sh->n_local = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (key[i] != ~0ull) local[atomicAdd(&sh->n_local, 1u)] = key[i];
        cl.sync();
    }

    // The token at which the running sum of the weights, over the cluster in the order of
    // the indexes, passes pick_of_total(total); f(d, index, w) sets the weights w of four
    // tokens from `index` on, and the thread that holds the token calls found(index, w, total).
    template <typename F, typename P, typename G>
    TMAC_DEV void draw(F&& f, P&& pick_of_total, G&& found)
    {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int n_chunks = (vectors() + L::kChunkVecs - 1) / L::kChunkVecs;
        unsigned long long mine = 0, all, total = 0, before = 0;
        for (int c = warp; c < n_chunks; c += kWarps) {
            unsigned long long s = 0;
            vectors(c * L::kChunkVecs + lane, min(vectors(), (c + 1) * L::kChunkVecs), 32, [&](const float (&e)[4], int j) {
                unsigned long long w[4];
                f(e, begin + j, w);
                s += (w[0] + w[1]) + (w[2] + w[3]);
            });
            s = warp_sum(s);
            if (lane == 0) chunks[c] = s;
            mine += s;
        }
        block_scan(lane == 0 ? mine : 0, sh->red_w, &all);
        if (threadIdx.x == 0) sh->kept = all;
        cl.sync();
        for (int r = 0; r < ranks; r++) {
            const unsigned long long w = cl.map_shared_rank(sh, r)->kept;
            total += w;
            if (r < rank) before += w;
        }
        const unsigned long long pick = pick_of_total(total);
        if (before <= pick && pick < before + all) {  // the whole CTA
            unsigned long long sum;
            for (int c0 = 0; c0 < n_chunks; c0 += kThreads) {
                const int c = c0 + threadIdx.x;
                const unsigned long long s = c < n_chunks ? chunks[c] : 0, at = before + block_scan(s, sh->red_w, &sum);
                if (at <= pick && pick < at + s) {
                    sh->chunk = c;
                    sh->chunk_before = at;
                }
                before += sum;
            }
            __syncthreads();
            const int v = sh->chunk * L::kChunkVecs + threadIdx.x;
            unsigned long long w[4] = {};
            if (threadIdx.x < L::kChunkVecs && v < vectors()) {
                const float4 q = load4(v);
                const float e[4] = {d_of(q.x), d_of(q.y), d_of(q.z), d_of(q.w)};
                f(e, begin + 4 * v - pad, w);
            }
            unsigned long long at = sh->chunk_before + block_scan(w[0] + w[1] + w[2] + w[3], sh->red_w, &sum);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (at <= pick && pick < at + w[i]) found(begin + 4 * v - pad + i, w[i], total);
                at += w[i];
            }
        }
        cl.sync();  // no CTA goes on while another reads its shared memory
    }
    // The index of the m-th element (from 1) with bits(d) == key, over the cluster.
    TMAC_DEV int tie(uint32_t key, uint32_t m)
    {
        draw(
            [&](const float (&e)[4], int, unsigned long long (&w)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = __float_as_uint(e[i]) == key;
            },
            [&](unsigned long long) { return m - 1; },
             [&](int index, unsigned long long, unsigned long long) {
                 for (int r = 0; r < ranks; r++) cl.map_shared_rank(sh, r)->tie_index = index;
             });
        return sh->tie_index;
    }

    // The number of the cluster's listed tokens, or -1 if they do not fit in one CTA;
    // this rank's come after `offset`.
    TMAC_DEV int listed(uint32_t* offset) const
    {
        const int lane = threadIdx.x & 31;
        const uint32_t c = lane < ranks ? cl.map_shared_rank(sh, lane)->n_local : 0, up = warp_scan(c);
        const uint32_t all = __shfl_sync(0xffffffffu, up, 31);
        *offset = __shfl_sync(0xffffffffu, up - c, rank);
        return __any_sync(0xffffffffu, c > (uint32_t)L::kLocal) || all > kList ? -1 : (int)all;
    }
    // Copies every rank's listed tokens into this CTA's keys.
    TMAC_DEV void gather() const
    {
        const int lane = threadIdx.x & 31;
        const uint32_t c = lane < ranks ? cl.map_shared_rank(sh, lane)->n_local : 0, up = warp_scan(c);
        for (int r = 0; r < ranks; r++) {  // a warp to a rank, or several
            const uint32_t count = __shfl_sync(0xffffffffu, c, r), at = __shfl_sync(0xffffffffu, up - c, r);
            const unsigned long long* from = cl.map_shared_rank(local, r);
            const int part = kWarps / ranks, warp = threadIdx.x >> 5;
            if (warp / part == r)
                for (uint32_t i = warp % part * 32 + lane; i < count; i += part * 32) sh->key[at + i] = from[i];
        }
        __syncthreads();
    }

    // Sums the weights (and with kCounts the numbers) of the elements for which bin_of gives a bin.
    template <bool kCounts, typename F>
    TMAC_DEV void histogram(F&& bin_of)
    {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh->cnt[i] = sh->hi[i] = sh->lo[i] = 0;
        __syncthreads();
        vectors(threadIdx.x, vectors(), kThreads, [&](const float (&e)[4], int) {
            // the four side by side: weights, then additions
            unsigned long long w[4];
            uint32_t old[4];
            int b[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[i] = weight_of(weight_exp(e[i]));
                b[i] = w[i] ? bin_of(e[i]) : -1;
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (b[i] < 0) continue;
                if (kCounts) atomicAdd(&sh->cnt[b[i]], 1u);
                old[i] = atomicAdd(&sh->lo[b[i]], (uint32_t)w[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (b[i] >= 0) add_carry(b[i], w[i], old[i]);
        });
        cl.sync();
        // this rank's share of the bins, over all ranks: `each` threads to a bin
        const int share = kBins / ranks, each = kThreads / share;
        uint32_t c_sum = 0;
        unsigned long long w_sum = 0;
        const int bin = threadIdx.x / each, part = threadIdx.x % each;
        for (int r = part; r < ranks; r += each) {
            const Shared* o = cl.map_shared_rank(sh, r);
            c_sum += o->cnt[rank * share + bin];
            w_sum += ((unsigned long long)o->hi[rank * share + bin] << 32) + o->lo[rank * share + bin];
        }
        for (int o = each / 2; o > 0; o >>= 1) {
            c_sum += __shfl_xor_sync(0xffffffffu, c_sum, o);
            w_sum += __shfl_xor_sync(0xffffffffu, w_sum, o);
        }
        if (part == 0) {
            sh->mcnt[bin] = c_sum;
            sh->mw[bin] = w_sum;
        } else {
            c_sum = 0;
            w_sum = 0;
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
                    c += o->mcnt[lane * per + i];
                    w += o->mw[lane * per + i];
                }
                up_c = base_c + warp_scan(c);
                up_w = base_w + warp_scan(w);
                hit = __ballot_sync(0xffffffffu, reached(up_c, up_w));
                if (lane == __ffs(hit) - 1) {
                    c = up_c - c;
                    w = up_w - w;
                    for (int i = lane * per;; i++) {
                        const uint32_t bc = o->mcnt[i];
                        const unsigned long long bw = o->mw[i];
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

    // Cuts the order after its first k elements (k > 0), or after the element at which
    // the running weight reaches p times the weight of the row (or of `of`, if not 0).
    // Elements of weight 0 do not count.
    TMAC_DEV Cut select(uint32_t k, float p, unsigned long long of)
    {
        Cut cut;
        if (k)
            histogram<true>([](float v) { return first_bin(v); });
        else
            histogram<false>([](float v) { return first_bin(v); });
        const int lane = threadIdx.x & 31;
        const unsigned long long row_w = warp_sum(lane < ranks ? cl.map_shared_rank(sh, lane)->share_w : 0);
        const double t = __dmul_rn((double)p, (double)(of ? of : row_w));
        if (!search(k, t, 0, 0)) {  // fewer than k: all of them
            cut.weight = row_w;
            return cut;
        }
        cut.set_bin(sh->found_bin);
        uint32_t found_c = sh->found_c, before_c = sh->before_c;
        unsigned long long found_w = sh->found_w, before_w = sh->before_w;
        list(cut.from, cut.to, [&](float v) { return first_bin(v) == cut.bin; });
        uint32_t offset;
        const int n = listed(&offset);
        if (n >= 0) {
            gather();
            cut_list(n, cut.from, cut.to, k ? k - before_c : 0, t, before_w);
            cl.sync();  // the lists are free again
            cut.last = sh->cut_key;
            cut.weight = sh->cut_weight;
            return cut;
        }
        uint32_t lo = __float_as_uint(cut.from), span = __float_as_uint(cut.to) - lo + 1;
        while (true) {
            int shift = 0;
            while ((span - 1) >> shift >= kBins) shift++;
            histogram<true>([&](float v) {
                const uint32_t o = __float_as_uint(v) - lo;
                return first_bin(v) == cut.bin && o < span ? (int)(o >> shift) : -1;
            });
            if (!search(k, t, before_c, before_w)) return cut;  // cannot happen: the bin holds the cut
            lo += (uint32_t)sh->found_bin << shift;
            span = 1u << shift;
            found_c = sh->found_c;
            before_c = sh->before_c;
            found_w = sh->found_w;
            before_w = sh->before_w;
            if (found_c == 1 || (k && before_c + found_c == k) || span == 1) break;
            __syncthreads();  // every thread has read the search
        }
        uint32_t m = found_c;
        if (span == 1) {  // equal ones: the first m of them
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
            found_w = m * each;
        }
        cut.weight = before_w + found_w;
        cut.last = (unsigned long long)(lo + span - 1) << 32 | 0xFFFFFFFFu;
        if (m < found_c) cut.last = (unsigned long long)lo << 32 | (uint32_t)tie(lo, m);
        return cut;
    }

    // Cuts the n gathered tokens, with d from `from` to `to`, after their first k (k >
    // 0), or where base plus their running weight reaches t: cut_key, and cut_weight
    // with base.  Many are first narrowed to the one of kBins parts that holds the cut.
    TMAC_DEV void cut_list(int n, float from, float to, uint32_t k, double t, unsigned long long base)
    {
        if (n > kFew) {
            const float scale = __fdiv_rn((float)(kBins - 1), __fsub_rn(to, from));
            const auto part_of = [&](unsigned long long key) {
                return min(max((int)__fmul_rn(__fsub_rn(__uint_as_float((uint32_t)(key >> 32)), from), scale), 0), kBins - 1);
            };
            for (int i = threadIdx.x; i < kBins; i += kThreads) sh->cnt[i] = sh->hi[i] = sh->lo[i] = 0;
            if (threadIdx.x == 0) sh->n_few = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += kThreads) {
                const int part = part_of(sh->key[i]);
                add_weight(part, weight_of(weight_exp(__uint_as_float((uint32_t)(sh->key[i] >> 32)))));
                atomicAdd(&sh->cnt[part], 1u);
            }
            __syncthreads();
            // a part to a thread
            unsigned long long all;
            const uint32_t c = threadIdx.x < kBins ? sh->cnt[threadIdx.x] : 0;
            const unsigned long long w = threadIdx.x < kBins ? ((unsigned long long)sh->hi[threadIdx.x] << 32) + sh->lo[threadIdx.x] : 0;
            const uint32_t before_c = (uint32_t)block_scan(c, sh->red_w, &all);
            const unsigned long long before_w = base + block_scan(w, sh->red_w, &all);
            if (k ? before_c < k && k <= before_c + c : (double)before_w < t && (double)(before_w + w) >= t) {
                sh->found_bin = threadIdx.x;
                sh->before_c = before_c;
                sh->before_w = before_w;
            }
            __syncthreads();
            const int part = sh->found_bin;
            for (int i = threadIdx.x; i < n; i += kThreads)
                if (part_of(sh->key[i]) == part) {
                    const uint32_t at = atomicAdd(&sh->n_few, 1u);
                    if (at < kFew) sh->pairs[at] = sh->key[i];
                }
            __syncthreads();
            if (sh->n_few <= kFew) {
                n = (int)sh->n_few;
                if (k) k -= sh->before_c;
                base = sh->before_w;
                if ((int)threadIdx.x < n) sh->key[threadIdx.x] = sh->pairs[threadIdx.x];
                __syncthreads();
            }
        }
        if (n <= kFew) {
            const unsigned long long mine = (int)threadIdx.x < n ? sh->key[threadIdx.x] : ~0ull;
            const unsigned long long w = (int)threadIdx.x < n ? weight_of(weight_exp(__uint_as_float((uint32_t)(mine >> 32)))) : 0;
            unsigned long long before;
            int rank;
            count_before(sh->pairs, n, mine, w, &rank, &before);
            before += base;
            if ((int)threadIdx.x < n && (k ? rank == (int)k - 1 : (double)before < t && (double)(before + w) >= t)) {
                sh->cut_key = mine;
                sh->cut_weight = before + w;
            }
            __syncthreads();
            return;
        }
        sort_and_cut(n, k, t, base);
    }
    TMAC_DEV void add_weight(int bin, unsigned long long w)
    {
        add_carry(bin, w, atomicAdd(&sh->lo[bin], (uint32_t)w));
    }
    // The upper word of an addition to a bin whose lower word was `old`.
    TMAC_DEV void add_carry(int bin, unsigned long long w, uint32_t old)
    {
        const uint32_t carry = old > 0xFFFFFFFFu - (uint32_t)w;
        if (carry + (w >> 32)) atomicAdd(&sh->hi[bin], carry + (uint32_t)(w >> 32));
    }
    TMAC_DEV void sort_and_cut(int n, uint32_t k, double t, unsigned long long base)
    {
        constexpr int kPer = kList / kThreads;
        sort_keys(sh->key, n);
        unsigned long long w[kPer], sum = 0, all;
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = threadIdx.x * kPer + i;
            w[i] = at < n ? weight_of(weight_exp(__uint_as_float((uint32_t)(sh->key[at] >> 32)))) : 0;
            sum += w[i];
        }
        unsigned long long before = base + block_scan(sum, sh->red_w, &all);
#pragma unroll
        for (int i = 0; i < kPer; i++) {
            const int at = threadIdx.x * kPer + i;
            const bool last = k ? at == (int)k - 1 : (double)before < t && (double)(before + w[i]) >= t;
            if (at < n && last) {
                sh->cut_key = sh->key[at];
                sh->cut_weight = before + w[i];
            }
            before += w[i];
        }
        __syncthreads();
    }
};

// The cuts and the draw over the n gathered tokens, the first k of the order among them.
TMAC_DEV void draw_from_list(const SampleArgs& a, Shared* sh, int b, int n, int k, float p, float m)
{
    unsigned long long* key = sh->key;
    if (n <= kFew) {
        __syncthreads();
        const unsigned long long mine = (int)threadIdx.x < n ? key[threadIdx.x] : ~0ull;
        const float e = (int)threadIdx.x < n ? weight_exp(__uint_as_float((uint32_t)(mine >> 32))) : 0.0f;
        unsigned long long w = (int)threadIdx.x < n ? weight_of(e) : 0, before;
        int rank;
        count_before(sh->pairs, n, mine, w, &rank, &before);
        bool kept = (int)threadIdx.x < n && rank < k;
        if (p < 1.0f) {
            const unsigned long long all = sum_few(kept ? w : 0, n, sh->red_w);
            kept = kept && ((double)before < __dmul_rn((double)p, (double)all) || rank == 0);
        }
        kept = kept && (e >= m || rank == 0);
        if (!kept) w = 0;
        const unsigned long long all = sum_few(w, n, sh->red_w), pick = pick_of(a.u[b], all);
        count_before(sh->pairs, n, mine & 0xFFFFFFFFu, w, &rank, &before);  // in the order of the indexes
        if (before <= pick && pick < before + w) {
            a.tokens[b] = (int)(uint32_t)mine;
            a.probs[b] = (float)__ddiv_rn((double)w, (double)all);
        }
        return;
    }
    constexpr int kPer = kList / kThreads;
    if (threadIdx.x == 0) sh->n_keep = 1;
    sort_keys(key, n);
    const int n_k = min(k, n);
    float e[kPer];
    unsigned long long w[kPer], sum = 0, all;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int at = threadIdx.x * kPer + i;
        e[i] = at < n_k ? weight_exp(__uint_as_float((uint32_t)(key[at] >> 32))) : 0.0f;
        w[i] = at < n_k ? weight_of(e[i]) : 0;
        sum += w[i];
    }
    unsigned long long before = block_scan(sum, sh->red_w, &all);
    const double t = __dmul_rn((double)p, (double)all);
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
    const int kept = (int)sh->n_keep;

    // the kept ones in the order of their indexes
    for (int i = threadIdx.x; i < kept; i += kThreads) key[i] = key[i] << 32 | key[i] >> 32;
    sort_keys(key, kept);
    sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int at = threadIdx.x * kPer + i;
        w[i] = at < kept ? weight_of(weight_exp(__uint_as_float((uint32_t)key[at]))) : 0;
        sum += w[i];
    }
    before = block_scan(sum, sh->red_w, &all);
    const unsigned long long pick = pick_of(a.u[b], all);
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        if (before <= pick && pick < before + w[i]) {
            a.tokens[b] = (int)(key[threadIdx.x * kPer + i] >> 32);
            a.probs[b] = (float)__ddiv_rn((double)w[i], (double)all);
        }
        before += w[i];
    }
}

// l * inv of the CTA's n logits into x, NaN as -inf, and `pad` (and up to 3 more
// behind) -inf around them; the largest of the thread's.
template <typename T>
TMAC_DEV float load_scaled(const T* l, int n, float inv, float* x, int pad)
{
    float mx = -INFINITY;
    auto put = [&](int i) {
        x[i] = fmaxf(__fmul_rn(Elem<T>::load(l + i), inv), -INFINITY);  // fmaxf leaves a NaN out
        mx = fmaxf(mx, x[i]);
    };
    constexpr int kVec = 16 / sizeof(T), kFlight = 4;
    const int head = min(n, (int)((16 - (uintptr_t)l % 16) % 16 / sizeof(T)));
    const int vecs = (n - head) / kVec, tail = head + vecs * kVec;
    if ((int)threadIdx.x < head) put(threadIdx.x);
    if ((int)threadIdx.x < n - tail) put(tail + threadIdx.x);
    if ((int)threadIdx.x < pad) x[-1 - (int)threadIdx.x] = -INFINITY;
    if ((int)threadIdx.x < 3) x[n + threadIdx.x] = -INFINITY;
    const uint4* v = reinterpret_cast<const uint4*>(l + head);
    for (int i0 = threadIdx.x; i0 < vecs; i0 += kThreads * kFlight) {
        uint4 r[kFlight];
#pragma unroll
        for (int f = 0; f < kFlight; f++)
            if (i0 + f * kThreads < vecs) r[f] = __ldg(v + i0 + f * kThreads);
#pragma unroll
        for (int f = 0; f < kFlight; f++) {
            if (i0 + f * kThreads >= vecs) break;
            T in[kVec];
            *reinterpret_cast<uint4*>(in) = r[f];
            float4 y[kVec / 4];
            float* yf = reinterpret_cast<float*>(y);
#pragma unroll
            for (int c = 0; c < kVec; c++) {
                yf[c] = fmaxf(__fmul_rn(Elem<T>::load(in + c), inv), -INFINITY);
                mx = fmaxf(mx, yf[c]);
            }
#pragma unroll
            for (int c = 0; c < kVec / 4; c++)
                *reinterpret_cast<float4*>(x + head + (i0 + f * kThreads) * kVec + 4 * c) = y[c];
        }
    }
    return mx;
}

template <typename T, bool kResident>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    using R = Row<T, kResident>;
    R row = {cg::this_cluster()};
    Shared* sh = row.sh = reinterpret_cast<Shared*>(smem);
    row.local = reinterpret_cast<unsigned long long*>(smem + kSharedBytes);
    row.chunks = row.local + R::L::kLocal;
    row.ranks = (int)row.cl.num_blocks();
    row.rank = (int)row.cl.block_rank();
    const int b = blockIdx.x / row.ranks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    row.begin = row.rank * a.slice;
    row.n = max(0, min(a.slice, a.vocab - row.begin));
    row.l = (const T*)a.logits + b * a.stride + row.begin;
    // vectors of 4 logits start on a multiple of their size; so do those of x
    row.pad = (int)((uintptr_t)row.l % (4 * sizeof(T)) / sizeof(T));
    row.x = reinterpret_cast<float*>(smem + list_bytes<kResident>()) + row.pad;
    row.infinite = false;

    const float temperature = a.temperature ? a.temperature[b] : 1.0f;
    const float inv = __frcp_rn(temperature);
    const bool greedy = !(temperature > 0.0f) || isinf(inv);
    row.inv = greedy ? 1.0f : inv;
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
    float own_max = -INFINITY, least = INFINITY;
    if (kResident) {
        own_max = load_scaled<T>(row.l, row.n, row.inv, row.x, row.pad);
    } else if (row.mx = 0.0f; k > 1 && !greedy) {
        own_max = row.max_and_list((uint32_t)k, &least);
        __syncthreads();  // the maxima's counts have been read
    } else {
        row.vectors(threadIdx.x, row.vectors(), kThreads, [&](const float (&e)[4], int) {  // here -x
            own_max = fmaxf(own_max, -fminf(fminf(e[0], e[1]), fminf(e[2], e[3])));
        });
    }
    float mx = own_max;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) sh->red_f[warp] = mx;
    if (threadIdx.x < R::L::kSteps) sh->maxima[threadIdx.x] = 0;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWarps; i++) mx = fmaxf(mx, sh->red_f[i]);
        sh->cta_max = mx;
        sh->least = least < INFINITY && sh->n_local <= R::L::kLocal ? least : INFINITY;
    }
    row.cl.sync();
    mx = lane < row.ranks ? row.cl.map_shared_rank(sh, lane)->cta_max : -INFINITY;
    for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = row.mx = __fadd_rn(__shfl_sync(0xffffffffu, mx, 0), 0.0f);  // -0 as 0: no d is -0
    row.infinite = mx == INFINITY;
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
        row.vectors(threadIdx.x, row.vectors(), kThreads, [&](const float (&e)[4], int j) {
#pragma unroll
            for (int c = 3; c >= 0; c--)
                if (e[c] == 0.0f) first = min(first, row.begin + j + c);
        });
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

    Cut cut;
    if (k > 0) {
        // the least bound on d below which k threads have their maximum
        row.count_maximum(row.d_of(own_max));
        row.cl.sync();
        const float bound = R::bound_of((uint32_t)k, [&] {
            typename R::Counts sum = {};
#pragma unroll 8
            for (int r = 0; r < row.ranks; r++) {
                const auto c = reinterpret_cast<const typename R::Counts*>(row.cl.map_shared_rank(sh, r)->maxima)[lane];
#pragma unroll
                for (int i = 0; i < R::kMine; i++) reinterpret_cast<uint32_t*>(&sum)[i] += reinterpret_cast<const uint32_t*>(&c)[i];
            }
            return sum;
        });
        if (bound < INFINITY) {
            // Tokens that a rank has not listed lie at least as far as its `least`.
            bool all_listed = !kResident;
            if (!kResident) {
                const float far = lane < row.ranks ? row.d_of(row.cl.map_shared_rank(sh, lane)->least) : INFINITY;
                all_listed = __all_sync(0xffffffffu, far >= bound);
            }
            if (all_listed)
                row.relist(bound);
            else
                row.list(0.0f, bound, [](float) { return true; });
            uint32_t offset;
            const int n = row.listed(&offset);
            if (n >= 0) {
                Shared* first = row.cl.map_shared_rank(sh, 0);
                for (uint32_t i = threadIdx.x; i < sh->n_local; i += kThreads) first->key[offset + i] = row.local[i];
                row.cl.sync();
                if (row.rank == 0) draw_from_list(a, sh, b, n, k, p, m);
                return;  // nobody reads another CTA's shared memory any more
            }
            row.cl.sync();  // the others have read this CTA's count
        }
        cut = row.select((uint32_t)k, 0.0f, 0);
    }
    if (p < 1.0f) {
        __syncthreads();
        cut = row.select(0, p, cut.weight);
    }

    // the draw, in the order of the indexes
    const auto pick = [&](unsigned long long total) { return pick_of(a.u[b], total); };
    const auto found = [&](int index, unsigned long long w, unsigned long long total) {
        a.tokens[b] = index;
        a.probs[b] = (float)__ddiv_rn((double)w, (double)total);
    };
    // no kept token lies as far: a bound on exp(-d) >= m, a little wide, and on the cut
    const float farthest = fminf(cut.to, m > 0.0f ? __fadd_rn(__fmul_rn(-logf(m), 1.0001f), 1e-4f) : INFINITY);
    if (cut.last == ~0ull && m == 0.0f)
        row.draw(
            [](const float (&d)[4], int, unsigned long long (&w)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = weight_of(weight_exp(d[i]));
            },
            pick, found);
    else
        row.draw(
            [&](const float (&d)[4], int index, unsigned long long (&w)[4]) {
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = 0;
                // Read anew, or by min-p, most vectors have no token near enough; others are
                // worked on side by side (top-p of 32 held rows 39 us, 43 with the test).
                if ((!kResident || m > 0.0f) && !(fminf(fminf(d[0], d[1]), fminf(d[2], d[3])) < farthest)) return;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float e = weight_exp(d[i]);
                    w[i] = order_key(d[i], index + i) <= cut.last && e >= m ? weight_of(e) : 0;
                }
            },
            pick, found);
}

template <typename T, bool kResident>
int launch_sample(const SampleArgs& a, int batch, int ranks, int device, cudaStream_t s)
{
    const size_t smem = sample_bytes<kResident>(a.slice);
    auto fn = sample_kernel<T, kResident>;
    static std::atomic<uint64_t> done{0};
    const int rc = set_once(done, device, [&] {
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        return e ? e : cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (rc) return rc;
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
    if (vocab <= 0 || vocab > kMaxVocab) return fail(TMAC_ERR_SHAPE, "vocab must be 1 to 720000");
    if (batch > 1 && row_stride && row_stride < vocab) return fail(TMAC_ERR_SHAPE, "row_stride must cover a row");
    if (device < 0) return fail(TMAC_ERR_NODEV, "no such CUDA device");
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
    // Up to two CTAs per SM hold their rows; more rows than that are read anew for
    // each pass by as few CTAs as fill the SMs twice.  Top-k 40 of 151936 logits, held
    // against read anew: 15.4 / 25.0 us for 32 rows, 36.2 / 18.0 for 64, 126 / 40 for 256.
    // So are more rows of fewer logits: what half an SM's shared memory holds.
    const int room = 2 * num_sms(device), most = vocab <= 4096 ? 1 : vocab <= kCluster * kMaxSlice ? kCluster : kMaxCluster;
    int ranks = most;
    while (ranks > 1 && (int64_t)batch * ranks > room) ranks /= 2;
    a.slice = ((vocab + ranks - 1) / ranks + 7) & ~7;  // every rank's first logit is as aligned as the row's
    const bool resident = (int64_t)batch * ranks <= room && (ranks == most || sample_bytes<true>(a.slice) <= 113 * 1024);
    DeviceGuard dg(device);
    if (!dg.ok) return fail(TMAC_ERR_NODEV, "no such CUDA device");
    return with_type(type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return resident ? launch_sample<T, true>(a, batch, ranks, device, (cudaStream_t)stream)
                        : launch_sample<T, false>(a, batch, ranks, device, (cudaStream_t)stream);
    });
}
