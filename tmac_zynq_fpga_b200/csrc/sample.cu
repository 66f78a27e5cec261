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
// One cluster of CTAs per row holds the row's d in shared memory.  The cut of
// top-k / top-p is found by radix selection on the bits of d: a 2048-bin
// histogram of counts and weights per round, at most four rounds, each bin
// summed over the cluster through distributed shared memory.
//
// Bound: HBM for large batches (every logit is read once), latency for one row.
#include "serving.cuh"

#include <cooperative_groups.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace tmac {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kBins = 2048;
constexpr float kBinScale = 91.0f;     // bins per unit of d in the first round; d < 22.2 where w > 0
constexpr int kMaxCluster = 16, kMaxSlice = 45000;

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
    uint32_t cnt[kBins], hi[kBins], lo[kBins];  // this CTA's histogram: counts, weights in two halves
    uint32_t mcnt[kBins];                       // this CTA's share of the bins, summed over the cluster
    unsigned long long mw[kBins];
    unsigned long long share_w, red_w[kWarps];
    uint32_t share_c, red_c[kWarps];
    float red_f[kWarps], cta_max;
    int cta_min_index;
    uint32_t tie_count;
    unsigned long long kept;
    // broadcast of a search
    int found_bin, tie_index;
    uint32_t found_c, before_c;
    unsigned long long found_w, before_w;
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
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh->cnt[i] = sh->hi[i] = sh->lo[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float v = d[i];
            const unsigned long long w = weight_of(weight_exp(v));
            if (!w) continue;
            const int b = bin_of(v);
            if (b < 0) continue;
            // a slice has at most kMaxSlice elements of at most 2^16 in either half: no overflow
            atomicAdd(&sh->cnt[b], 1u);
            atomicAdd(&sh->hi[b], (uint32_t)(w >> 16));
            atomicAdd(&sh->lo[b], (uint32_t)(w & 0xFFFF));
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
                c += o->cnt[rank * share + i];
                w += ((unsigned long long)o->hi[rank * share + i] << 16) + o->lo[rank * share + i];
            }
            sh->mcnt[i] = c;
            sh->mw[i] = w;
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
    TMAC_DEV bool search(uint32_t k, double t, uint32_t base_c, unsigned long long base_w)
    {
        if (threadIdx.x == 0) {
            sh->found_bin = -1;
            uint32_t c = base_c;
            unsigned long long w = base_w;
            const int share = kBins / ranks;
            for (int r = 0; r < ranks && sh->found_bin < 0; r++) {
                const Shared* o = cl.map_shared_rank(sh, r);
                const uint32_t rc = o->share_c;
                const unsigned long long rw = o->share_w;
                if (k ? c + rc < k : (double)(w + rw) < t) {
                    c += rc;
                    w += rw;
                    continue;
                }
                for (int i = 0; i < share; i++) {
                    const uint32_t bc = o->mcnt[i];
                    const unsigned long long bw = o->mw[i];
                    if (k ? c + bc >= k : (double)(w + bw) >= t) {
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

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(SampleArgs a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    Row row = {cg::this_cluster()};
    row.sh = reinterpret_cast<Shared*>(smem);
    row.d = reinterpret_cast<float*>(smem + sizeof(Shared));
    row.ranks = (int)row.cl.num_blocks();
    row.rank = (int)row.cl.block_rank();
    Shared* sh = row.sh;
    const int b = blockIdx.x / row.ranks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    row.begin = row.rank * a.slice;
    row.n = max(0, min(a.slice, a.vocab - row.begin));

    const float temperature = a.temperature ? a.temperature[b] : 1.0f;
    float inv = __frcp_rn(temperature);
    const bool greedy = !(temperature > 0.0f) || isinf(inv);
    if (greedy) inv = 1.0f;

    // scaled logits, and the largest of the row
    const T* l = (const T*)a.logits + b * a.stride + row.begin;
    float mx = -INFINITY;
    for (int i = threadIdx.x; i < row.n; i += kThreads) {
        float x = __fmul_rn(Elem<T>::load(l + i), inv);
        if (isnan(x)) x = -INFINITY;
        row.d[i] = x;
        mx = fmaxf(mx, x);
    }
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) sh->red_f[warp] = mx;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kWarps; i++) mx = fmaxf(mx, sh->red_f[i]);
        sh->cta_max = mx;
    }
    row.cl.sync();
    mx = -INFINITY;
    for (int r = 0; r < row.ranks; r++) mx = fmaxf(mx, row.cl.map_shared_rank(sh, r)->cta_max);
    if (mx == -INFINITY) {  // nothing to choose from
        row.cl.sync();
        if (row.rank == 0 && threadIdx.x == 0) {
            a.tokens[b] = -1;
            a.probs[b] = 0.0f;
        }
        return;
    }
    int first = 0x7FFFFFFF;  // lowest index of the largest
    for (int i = threadIdx.x; i < row.n; i += kThreads) {
        const float x = row.d[i];
        row.d[i] = x == mx ? 0.0f : __fsub_rn(mx, x);
        if (x == mx) first = min(first, row.begin + i);
    }

    int k = a.top_k ? a.top_k[b] : 0;
    if (k < 0 || k >= a.vocab) k = 0;
    const float p = a.top_p ? a.top_p[b] : 1.0f;
    float m = a.min_p ? a.min_p[b] : 0.0f;
    m = m > 0.0f ? fminf(m, 1.0f) : 0.0f;
    if (greedy || k == 1) {
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
    __syncthreads();

    Cut cut = {kBins, 0xFFFFFFFFu, 0x7FFFFFFF, 0};
    if (k > 0) cut = row.select((uint32_t)k, 0.0);
    if (p < 1.0f) {
        __syncthreads();
        if (p > 0.0f) {
            if (k <= 0) {  // the whole row's weight
                unsigned long long s = 0;
                for (int i = threadIdx.x; i < row.n; i += kThreads) s += weight_of(weight_exp(row.d[i]));
                s = warp_sum(s);
                if (lane == 0) sh->red_w[warp] = s;
                __syncthreads();
                if (threadIdx.x == 0) {
                    for (int i = 1; i < kWarps; i++) s += sh->red_w[i];
                    sh->kept = s;
                }
                row.cl.sync();
                for (int r = 0; r < row.ranks; r++) cut.weight += row.cl.map_shared_rank(sh, r)->kept;
                row.cl.sync();
            }
            cut = row.select(0, __dmul_rn((double)p, (double)cut.weight));
        } else {
            cut = row.select(1, 0.0);
        }
    }

    // the draw, in the order of the indexes
    auto kept_weight = [&](float v, int j, bool in) -> unsigned long long {
        if (!in || !kept_by(cut, v, row.begin + j)) return 0;
        const float e = weight_exp(v);
        return e >= m ? weight_of(e) : 0;
    };
    unsigned long long mine = 0;
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
    unsigned long long total = 0, before = 0;
    for (int r = 0; r < row.ranks; r++) {
        const unsigned long long w = row.cl.map_shared_rank(sh, r)->kept;
        total += w;
        if (r < row.rank) before += w;
    }
    for (int i = 0; i < warp; i++) before += sh->red_w[i];
    const double at = __dmul_rn((double)a.u[b], (double)total);
    unsigned long long pick = at > 0.0 ? (unsigned long long)at : 0;
    if (pick >= total) pick = total - 1;
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
    const size_t smem = sizeof(Shared) + (size_t)a.slice * sizeof(float);
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
    a.slice = (vocab + ranks - 1) / ranks;
    DeviceGuard dg(device);
    if (!dg.ok) return fail(TMAC_ERR_NODEV, "no such CUDA device");
    return with_type(type, [&](auto* t) {
        return launch_sample<std::remove_pointer_t<decltype(t)>>(a, batch, ranks, (cudaStream_t)stream);
    });
}
