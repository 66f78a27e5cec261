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
// head's group) against a range of 64-key tiles with a running maximum and sum; a
// job leaves (maximum, sum, unnormalised o), and attn_join_kernel joins a row's
// jobs.  Where that is less work than a second launch, every sequence reads the
// prefix itself, and one job holds all of a row's keys and writes its result.
//
// The products run on mma.sync with 32-bit sums.  16-bit elements are its operands
// as they are; a 32-bit one is split into the nearest tf32 number and the rest, cut to
// one, and three products of the parts make one of the elements but for 2^-21 of it.
// The tensor cores cut off what an addition to a sum loses, so products with a rest have
// a sum of their own, and sums of few products are added to the scores and to O by the
// FMA units.  The error against 64 bits is the plain form's, or up to half less (rms over
// 16384 keys of heads of 64 3.3e-8 and 3.2e-8, largest 7.6e-7 and 1.1e-6; sums over a whole
// head of 128 on the tensor cores had 1.4 times it, and took as long).  (Products on
// the FMA units too took 2 to 3 times as long.)  Tiles come through cp.async, several in
// flight.  The prefix's jobs of 16-bit elements go to the tcgen05 kernel of
// prefix_attention_tc.cu where there are rows enough.
//
// Bound: latency where there is little work: 48 sequences over 2051 + up to 509 keys (14/2
// heads of 64, f16) take 13.3 us, 10 of them jobs of 3 to 4 tiles, 3 the join; in 32 bits
// 25.2 us.  64 sequences with only their own keys (bf16, 14/2 heads of 64 and 16/4 of 128)
// run at 1900 and 3300 GB/s with 1024 each, at 3800 and 5100 with 8192.
#include "prefix_attention.cuh"

#include <cmath>

namespace tmac {
namespace {

TMAC_DEV void cp_async16(void* dst, const void* src, bool valid)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
TMAC_DEV void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
TMAC_DEV void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}
// Copies tiles of keys and values into shared memory, 16 bytes a thread.  A warp
// touches 16 keys of a tile; its lanes look their pages up one tile ahead of the
// copies, so a copy does not wait for a table.
template <typename T, int D>
struct Copier {
    static constexpr int kVec = 16 / sizeof(T), kPer = D / kVec;          // copies to a key
    static constexpr int kCopies = kTile * kPer / kThreads;               // of a thread
    static constexpr int kAtOnce = 32 / kPer < 1 ? 1 : 32 / kPer;         // keys of a warp's one copy
    static constexpr int kKeys = kTile / kWarps;                          // keys of the warp
    static_assert(kPer <= 32 && kKeys <= 32 && kKeys == kCopies * kAtOnce, "a lane to a key");
    // The tile's key that copy i of lane `lane` belongs to
    static TMAC_DEV int key_of(int i, int lane) { return (threadIdx.x >> 5) * kAtOnce + i * (kWarps * kAtOnce) + lane / kPer; }
    // The page of this lane's key in tile t
    static TMAC_DEV int look_up(const AttnArgs& a, const Job& j, int t)
    {
        const int lane = threadIdx.x & 31;
        if (t >= j.tile1 || lane >= kKeys) return 0;
        const TileOf tile = find_tile(a, j, t);
        const int g = tile.key0 + key_of(lane / kAtOnce, lane % kAtOnce * kPer);
        return g < tile.keys ? __ldg(tile.pages + (g >> a.cache.page_shift)) : 0;
    }
    // Starts tile t's copies, its look_up given; k_at(key, value) and v_at say where 16
    // bytes from that value on go.  Keys out of reach, and rows of a page outside the
    // pool (the error word says so), become zeros.
    template <typename FK, typename FV>
    static TMAC_DEV void start(const AttnArgs& a, const Job& j, int t, int page, FK&& k_at, FV&& v_at)
    {
        const int lane = threadIdx.x & 31, shift = a.cache.page_shift;
        const TileOf tile = find_tile(a, j, t);
        const bool known = page >= 0 && page < a.cache.n_pages;
        if (!known && lane < kKeys && tile.key0 + key_of(lane / kAtOnce, lane % kAtOnce * kPer) < tile.keys)
            record_error(a.err, TMAC_ERR_BOUNDS);
        const int safe = known ? page : -1;
#pragma unroll
        for (int i = 0; i < kCopies; i++) {
            const int key = key_of(i, lane), c = lane % kPer * kVec, g = tile.key0 + key;
            const int64_t pg = __shfl_sync(0xffffffffu, safe, i * kAtOnce + lane / kPer);
            const bool valid = pg >= 0 && g < tile.keys;
            const int64_t from = valid ? (((pg * a.cache.kv_heads + j.kvh) << shift) + (g & ((1 << shift) - 1))) * D + c : 0;
            cp_async16(k_at(key, c), (const T*)a.cache.k + from, valid);
            cp_async16(v_at(key, c), (const T*)a.cache.v + from, valid);
        }
    }
};
// ------------------------------------------------------------------ jobs ----
// Tiles of 16 rows per warp.  With up to 16 rows in the job the four warps take
// different 16 keys of a tile and join at the end; with more they take different rows.
// 16-bit weights are rounded to the elements' type for the second product, as the
// values are.  f16 has its 11 bits down to 2^-14 only: there the largest weight is 2^15,
// not 1, so that weights down to 2^-29 of it keep them and none above 2^-40 is lost.
constexpr int kMmaRows = 16, kStep = 16;
template <typename T>
constexpr float kLargestPower = std::is_same_v<T, __half> ? 15.0f : 0.0f;
template <typename T, int D>
struct MmaConf;
// 16-bit rows lie unpadded, their 16-byte pieces turned by the row's number: eight
// rows of one column fall on different banks.
template <typename T, int D>
struct MmaConf16 {
    static constexpr int kStages = D == 64 ? 4 : 3, kKeyRow = D, kValueRow = D;
    static constexpr int kWide = D == 64 ? 64 : 32;  // keys at a time where warps hold different rows
    static TMAC_DEV int key_at(int row, int c) { return row * D + ((c / 8 ^ (row & 7)) * 8 | c % 8); }
    static TMAC_DEV int value_at(int row, int c) { return key_at(row, c); }
};
template <int D>
struct MmaConf<__half, D> : MmaConf16<__half, D> {};
template <int D>
struct MmaConf<__nv_bfloat16, D> : MmaConf16<__nv_bfloat16, D> {};
// 32-bit rows are padded so that the fragments' loads fall on different banks.
template <int D>
struct MmaConf<float, D> {
    static constexpr int kStages = 3, kKeyRow = D + 8, kValueRow = D + 4;
    static constexpr int kWide = 16;  // 32 is no faster
    static TMAC_DEV int key_at(int row, int c) { return row * kKeyRow + c; }
    static TMAC_DEV int value_at(int row, int c) { return row * kValueRow + c; }
};
template <typename T, int D>
struct MmaSmem {
    struct {
        T k[kTile * MmaConf<T, D>::kKeyRow], v[kTile * MmaConf<T, D>::kValueRow];
    } stage[MmaConf<T, D>::kStages];
    float ml[kWarps][kMmaRows][2];
    uint32_t bad[kWarps][2];
};
TMAC_DEV void ldmatrix4(uint32_t (&r)[4], const void* p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}
TMAC_DEV void ldmatrix4_trans(uint32_t (&r)[4], const void* p)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}
template <typename T>
TMAC_DEV void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (std::is_same_v<T, __half>)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
TMAC_DEV void mma1688(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x as the nearest tf32 number and the rest (the product reads the upper 19 bits of
// each).  Nothing is added to the rest's bits: that of a NaN or an infinity is the NaN
// 0x7FFFFFFF, which an addition would turn into -0, and so would be lost where the
// addition above has turned x into -0 already.  A number that rounds to infinity has an
// infinite rest of the other sign.  Rows with such sums are computed again (row_by_keys).
TMAC_DEV void split_tf32(float x, uint32_t& hi, uint32_t& lo)
{
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(__fsub_rn(x, __uint_as_float(hi)));
}
// main += a b without the products of rests, which go to rest; a split already.
TMAC_DEV void mma_f32(float (&main)[4], float (&rest)[4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], float b0, float b1)
{
    uint32_t h0, l0, h1, l1;
    split_tf32(b0, h0, l0);
    split_tf32(b1, h1, l1);
    mma1688(rest, lo, h0, h1);
    mma1688(rest, hi, l0, l1);
    mma1688(main, hi, h0, h1);
}

template <typename T, int D>
TMAC_DEV void attn_mma(const AttnArgs& a)
{
    extern __shared__ __align__(16) uint8_t smem[];
    using Smem = MmaSmem<T, D>;
    using Conf = MmaConf<T, D>;
    Smem& sh = *reinterpret_cast<Smem*>(smem);
    constexpr bool k32 = sizeof(T) == 4;
    constexpr int kJobRows = kWarps * kMmaRows, kStages = Conf::kStages, kN = D / 8;
    constexpr int kDepth = k32 ? 8 : 16;  // of a product
    Job j;
    if (!find_job<kJobRows>(a, &j)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c2 = (lane & 3) * 2;
    const bool split_keys = j.rows <= kMmaRows;
    using Copy = Copier<T, D>;
    const auto copy = [&](int t, int page) {
        if (t < j.tile1) {
            auto& st = sh.stage[(t - j.tile0) % kStages];
            Copy::start(a, j, t, page, [&](int key, int c) { return &st.k[Conf::key_at(key, c)]; },
                        [&](int key, int c) { return &st.v[Conf::value_at(key, c)]; });
        }
        cp_async_commit();
    };
    int page[kStages];  // of the first tiles; then page[0], of the tile to copy next
#pragma unroll
    for (int i = 0; i < kStages; i++) page[i] = Copy::look_up(a, j, j.tile0 + i);

    // this thread's rows g and g + 8 of the warp's, as the product's first operand
    const int r0 = split_keys ? 0 : warp * kMmaRows;
    // (32 bits: depth t and t + 4 of a product are values 2 t and 2 t + 1, of Q and K alike)
    uint32_t q[D / kDepth][4];
    int p_limit[2], o_limit[2];
    const bool pairs = ((uintptr_t)a.q % (2 * sizeof(T)) | a.q_stride % 2) == 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = r0 + g + 8 * h;
        RowOf row = {0, 0, 0x7FFFFFFF, 0x7FFFFFFF};
        if (r < j.rows) row = find_row(a, j, r);
        p_limit[h] = row.p_limit;
        o_limit[h] = row.o_limit;
        const T* src = (const T*)a.q + row.token * a.q_stride + row.head * D + c2;
#pragma unroll
        for (int i = 0; i < D / 8; i++) {
            const T* at = src + 8 * i;
            if constexpr (k32) {
                float2 x = make_float2(0.0f, 0.0f);
                if (r < j.rows) x = pairs ? __ldg(reinterpret_cast<const float2*>(at)) : make_float2(at[0], at[1]);
                q[i][h] = __float_as_uint(x.x);
                q[i][2 + h] = __float_as_uint(x.y);
            } else {
                uint32_t x = 0;
                if (r < j.rows) {
                    if (pairs) {
                        x = __ldg(reinterpret_cast<const uint32_t*>(at));
                    } else {
                        const T two[2] = {at[0], at[1]};
                        x = *reinterpret_cast<const uint32_t*>(two);
                    }
                }
                q[i / 2][2 * (i % 2) + h] = x;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kStages - 1; i++) copy(j.tile0 + i, page[i]);
    page[0] = page[kStages - 1];
    // below these limits no row of the warp needs a mask
    const int p_least = __reduce_min_sync(0xffffffffu, min(p_limit[0], p_limit[1]));
    const int o_least = __reduce_min_sync(0xffffffffu, min(o_limit[0], o_limit[1]));
    const float scale = k32 ? a.scale : __fmul_rn(a.scale, 1.44269504f);  // log2 e: powers of 2
    float m[2], l[2], o[kN][4];
#pragma unroll
    for (int h = 0; h < 2; h++) m[h] = -INFINITY, l[h] = 0.0f;
#pragma unroll
    for (int n = 0; n < kN; n++)
#pragma unroll
        for (int c = 0; c < 4; c++) o[n][c] = 0.0f;

    for (int t = j.tile0; t < j.tile1; t++) {
        cp_async_wait<kStages - 2>();
        __syncthreads();
        copy(t + kStages - 1, page[0]);
        page[0] = Copy::look_up(a, j, t + kStages);
        const auto& st = sh.stage[(t - j.tile0) % kStages];
        const TileOf tile = find_tile(a, j, t);
        const int least = min(tile.prefix ? p_least : o_least, tile.keys);
        const int limits[2] = {min(tile.prefix ? p_limit[0] : o_limit[0], tile.keys), min(tile.prefix ? p_limit[1] : o_limit[1], tile.keys)};
        // kN8 * 8 keys from `step` on
        const auto keys = [&](auto n8, int step) {
            constexpr int kN8 = decltype(n8)::value;
            float s[kN8][4] = {};
            [[maybe_unused]] constexpr int kChain = 4;  // 32-bit products in a row on the tensor cores
            [[maybe_unused]] float main[k32 ? kN8 : 1][4] = {}, rest[k32 ? kN8 : 1][4] = {};
#pragma unroll
            for (int i = 0; i < D / kDepth; i++) {
                if constexpr (k32) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) split_tf32(__uint_as_float(q[i][c]), hi[c], lo[c]);
#pragma unroll
                    for (int n = 0; n < kN8; n++) {
                        const float2 kx = *reinterpret_cast<const float2*>(&st.k[Conf::key_at(step + 8 * n + g, 8 * i + c2)]);
                        mma_f32(main[n], rest[n], hi, lo, kx.x, kx.y);
                    }
                    if (i % kChain == kChain - 1)
#pragma unroll
                        for (int n = 0; n < kN8; n++)
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                s[n][c] = __fadd_rn(s[n][c], __fadd_rn(main[n][c], rest[n][c]));
                                main[n][c] = rest[n][c] = 0.0f;
                            }
                } else {
#pragma unroll
                    for (int n = 0; n < kN8; n += 2) {
                        uint32_t kx[4];  // keys 0-7 and 8-15, two halves of 16 dims each
                        ldmatrix4(kx, &st.k[Conf::key_at(step + 8 * n + (lane & 7) + (lane >> 4) * 8, 16 * i + (lane >> 3 & 1) * 8)]);
                        mma16816<T>(s[n], q[i], kx[0], kx[1]);
                        mma16816<T>(s[n + 1], q[i], kx[2], kx[3]);
                    }
                }
            }
            const bool some_masked = tile.key0 + step + 8 * kN8 > least;
            float al[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int limit = limits[h];
                float mx = -INFINITY;
#pragma unroll
                for (int n = 0; n < kN8; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float& x = s[n][2 * h + c];
                        x = __fmul_rn(x, scale);
                        if (some_masked && tile.key0 + step + 8 * n + c2 + c >= limit) x = -INFINITY;
                        mx = fmaxf(mx, x);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                mx = fmaxf(__fsub_rn(mx, kLargestPower<T>), m[h]);
                al[h] = mx == m[h] ? 1.0f : power<T>(__fsub_rn(m[h], mx));
                const float base = mx == -INFINITY ? 0.0f : mx;  // sees nothing yet: all 0
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < kN8; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float& x = s[n][2 * h + c];
                        x = power<T>(__fsub_rn(x, base));
                        sum = __fadd_rn(sum, x);
                    }
                m[h] = mx;
                l[h] = __fmaf_rn(l[h], al[h], sum);
            }
            if (__any_sync(0xffffffffu, al[0] != 1.0f || al[1] != 1.0f))
#pragma unroll
                for (int n = 0; n < kN; n++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[n][c] = __fmul_rn(o[n][c], al[c >> 1]);
            if constexpr (k32) {
                // depth t and t + 4: keys 2 t and 2 t + 1, as the scores lie
                uint32_t hi[kN8][4], lo[kN8][4];
#pragma unroll
                for (int k = 0; k < kN8; k++)
#pragma unroll
                    for (int c = 0; c < 4; c++) split_tf32(s[k][c >> 1 | (c & 1) << 1], hi[k][c], lo[k][c]);
#pragma unroll
                for (int n = 0; n < kN; n++) {
                    float sum[4] = {}, small[4] = {};
#pragma unroll
                    for (int k = 0; k < kN8; k++)
                        mma_f32(sum, small, hi[k], lo[k], st.v[Conf::value_at(step + 8 * k + c2, 8 * n + g)],
                                st.v[Conf::value_at(step + 8 * k + c2 + 1, 8 * n + g)]);
#pragma unroll
                    for (int c = 0; c < 4; c++) o[n][c] = __fadd_rn(o[n][c], __fadd_rn(sum[c], small[c]));
                }
            } else {
#pragma unroll
                for (int k = 0; k < kN8; k += 2) {
                    const uint32_t p[4] = {pack2<T>(s[k][0], s[k][1]), pack2<T>(s[k][2], s[k][3]), pack2<T>(s[k + 1][0], s[k + 1][1]),
                                           pack2<T>(s[k + 1][2], s[k + 1][3])};
#pragma unroll
                    for (int n = 0; n < kN; n += 2) {
                        uint32_t vx[4];  // keys 0-7 and 8-15 of dims 8n.., then of the next eight
                        ldmatrix4_trans(vx, &st.v[Conf::value_at(step + 8 * k + (lane & 15), 8 * n + (lane >> 4) * 8)]);
                        mma16816<T>(o[n], p, vx[0], vx[1]);
                        mma16816<T>(o[n + 1], p, vx[2], vx[3]);
                    }
                }
            }
        };
        if (split_keys) {
            if (tile.key0 + warp * kStep < tile.keys) keys(std::integral_constant<int, 2>(), warp * kStep);
        } else if (r0 < j.rows) {
            for (int step = 0; step < kTile && tile.key0 + step < tile.keys; step += Conf::kWide)
                keys(std::integral_constant<int, Conf::kWide / 8>(), step);
        }
    }
    cp_async_wait<0>();
    // Rows with a sum that is not finite are computed again (row_by_keys): bit 4 (r & 7) of
    // bad[r >> 3] for row r of the warp's.
    uint32_t bad[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        bool finite = true;
#pragma unroll
        for (int n = 0; n < kN; n++) finite &= fabsf(o[n][2 * h]) < INFINITY && fabsf(o[n][2 * h + 1]) < INFINITY;
        bad[h] = __ballot_sync(0xffffffffu, !finite);
        bad[h] |= bad[h] >> 1;
        bad[h] = (bad[h] | bad[h] >> 2) & 0x11111111u;
    }
    const auto is_bad = [](const uint32_t (&b)[2], int r) { return (b[r >> 3 & 1] >> (4 * (r & 7)) & 1) != 0; };
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l[h] = __fadd_rn(l[h], __shfl_xor_sync(0xffffffffu, l[h], 1));
        l[h] = __fadd_rn(l[h], __shfl_xor_sync(0xffffffffu, l[h], 2));
    }
    if (!split_keys) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = r0 + g + 8 * h;
            if (r >= j.rows || is_bad(bad, g + 8 * h)) continue;
            const RowOf row = find_row(a, j, r);
#pragma unroll
            for (int n = 0; n < kN; n++) {
                const float two[2] = {o[n][2 * h], o[n][2 * h + 1]};
                put_results<T, D, 2>(a, j, row, 8 * n + c2, m[h], l[h], two);
            }
        }
        if (bad[0] | bad[1])
            for (int r = 0; r < kMmaRows && r0 + r < j.rows; r++)
                if (is_bad(bad, r)) row_by_keys<T, D>(a, j, r0 + r);
        return;
    }
    // the warps' results, joined
    __syncthreads();
    float* ow = reinterpret_cast<float*>(&sh.stage[0]);  // [warps][16][D]
    static_assert(sizeof(float) * kWarps * kMmaRows * D <= sizeof(sh.stage), "join space");
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int r = g + 8 * h;
        if (c2 == 0) {
            sh.ml[warp][r][0] = m[h];
            sh.ml[warp][r][1] = l[h];
        }
#pragma unroll
        for (int n = 0; n < kN; n++)
            *reinterpret_cast<float2*>(&ow[(warp * kMmaRows + r) * D + 8 * n + c2]) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
        if (lane == 0) sh.bad[warp][h] = bad[h];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; h++) {
        bad[h] = 0;
#pragma unroll
        for (int w = 0; w < kWarps; w++) bad[h] |= sh.bad[w][h];
    }
    if (bad[0] | bad[1])
        for (int r = warp; r < j.rows; r += kWarps)
            if (is_bad(bad, r)) row_by_keys<T, D>(a, j, r);
    for (int i = threadIdx.x; i < j.rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (is_bad(bad, r)) continue;
        float mx = -INFINITY, sum = 0.0f, val[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWarps; w++) mx = fmaxf(mx, sh.ml[w][r][0]);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float lw = sh.ml[w][r][1];
            if (lw == 0.0f) continue;  // saw no key
            const float f = power<T>(__fsub_rn(sh.ml[w][r][0], mx));
            const float4 x = *reinterpret_cast<const float4*>(&ow[(w * kMmaRows + r) * D + d]);
            sum = __fmaf_rn(f, lw, sum);
            val[0] = __fmaf_rn(f, x.x, val[0]);
            val[1] = __fmaf_rn(f, x.y, val[1]);
            val[2] = __fmaf_rn(f, x.z, val[2]);
            val[3] = __fmaf_rn(f, x.w, val[3]);
        }
        put_results<T, D, 4>(a, j, find_row(a, j, r), d, mx, sum, val);
    }
}

// Jobs of an SM, by shared memory: the registers allow as many.
template <typename T, int D>
constexpr int kJobsOfSm = 227 * 1024 / (sizeof(MmaSmem<T, D>) + 1024);
template <typename T, int D>
__global__ void __launch_bounds__(kThreads, kJobsOfSm<T, D>) attn_mma_kernel(const __grid_constant__ AttnArgs a)
{
    attn_mma<T, D>(a);
    if (a.q_start && a.parts == 1) clear_rows<T, D, kWarps * kMmaRows>(a);
    // Where the tcgen05 kernel runs beside this one, this grid ends after it, so the
    // join, which waits for this grid, has waited for both.
    if (blockIdx.x == 0) pdl_wait();
}

// ------------------------------------------------------------------- join ----
// Joins the parts of one (token, head) per CTA: groups of D / 4 threads take every
// kGroups-th part, four values a thread, several loads in flight.
// Bound: latency and L2, 6 us for 1792 rows of 64 dims in 27 parts (12 MB).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) attn_join_kernel(AttnArgs a)
{
    constexpr int kLanes = D / 4, kGroups = kThreads / kLanes, kFlight = 4;
    __shared__ float weight[kThreads], red[kWarps][2];
    __shared__ float4 sums[kGroups][kLanes];
    const int64_t row = blockIdx.x;
    const int token = (int)(row / a.heads), head = (int)(row % a.heads);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = threadIdx.x / kLanes, d4 = threadIdx.x % kLanes;
    const int b = sequence_of(a, token);
    int n = 0;
    if (is_computed(a, token, b)) n = a.p_splits + (a.o_splits ? (tiles_of(own_len(a, b)) + a.o_range - 1) / a.o_range : 0);
    const float2* ml = a.part_ml + row * a.parts;
    const float4* po = reinterpret_cast<const float4*>(a.part_o + row * a.parts * D) + d4;
    pdl_wait();
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int s0 = 0; s0 < n; s0 += kThreads) {
        const int count = min(kThreads, n - s0);
        const float2 p = (int)threadIdx.x < count ? ml[s0 + threadIdx.x] : make_float2(-INFINITY, 0.0f);
        float mx = p.x;
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        if (lane == 0) red[warp][0] = mx;
        __syncthreads();
        mx = m;
#pragma unroll
        for (int w = 0; w < kWarps; w++) mx = fmaxf(mx, red[w][0]);
        // 0: saw no key; a NaN stays one, however little the part weighs
        const float f = p.y == 0.0f || p.y != p.y ? p.y : power<T>(__fsub_rn(p.x, mx));
        weight[threadIdx.x] = f;
        float sum = f == 0.0f ? 0.0f : __fmul_rn(f, p.y);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, w));
        if (lane == 0) red[warp][1] = sum;
        __syncthreads();
        const float al = m == mx ? 1.0f : power<T>(__fsub_rn(m, mx));
        m = mx;
        l = __fmul_rn(l, al);
#pragma unroll
        for (int w = 0; w < kWarps; w++) l = __fadd_rn(l, red[w][1]);
        o = make_float4(__fmul_rn(o.x, al), __fmul_rn(o.y, al), __fmul_rn(o.z, al), __fmul_rn(o.w, al));
        for (int s = group; s < count; s += kGroups * kFlight) {
            float4 v[kFlight];
            float g[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; u++) {
                const int at = s + u * kGroups;
                g[u] = at < count ? weight[at] : 0.0f;
                v[u] = at < count ? __ldg(po + (int64_t)(s0 + at) * kLanes) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int u = 0; u < kFlight; u++) {
                if (g[u] == 0.0f) continue;
                o.x = __fmaf_rn(g[u], v[u].x, o.x);
                o.y = __fmaf_rn(g[u], v[u].y, o.y);
                o.z = __fmaf_rn(g[u], v[u].z, o.z);
                o.w = __fmaf_rn(g[u], v[u].w, o.w);
            }
        }
        __syncthreads();
    }
    sums[group][d4] = o;
    __syncthreads();
    if (threadIdx.x < D) {
        float v = 0.0f;
#pragma unroll
        for (int g = 0; g < kGroups; g++) v = __fadd_rn(v, reinterpret_cast<const float*>(sums[g])[threadIdx.x]);
        Elem<T>::store((T*)a.out + token * a.out_stride + head * D + threadIdx.x, l == 0.0f ? 0.0f : __fdiv_rn(v, l));
    }
}

int jobs_of_sm(int type, int dim)
{
    if (type == TMAC_TYPE_F32) return dim == 64 ? kJobsOfSm<float, 64> : kJobsOfSm<float, 128>;
    return dim == 64 ? kJobsOfSm<__half, 64> : kJobsOfSm<__half, 128>;
}
// How the work is cut: key ranges so that the jobs of a kernel are about as many as
// the GPU holds at once, own parts counted as three quarters of their bound (they are
// ragged).  32-bit jobs take longer to a tile and are cut finer: at one wave of jobs 48
// sequences over 2051 keys took 30.7 us, at two and a half 25.2.
int plan(AttnArgs* a, int type, int sms)
{
    constexpr int job_rows = kWarps * kMmaRows;
    const int hk = a->cache.kv_heads, dim = a->cache.dim;
    const auto tiles = [](int keys) { return (int64_t)(keys + kTile - 1) / kTile; };
    const auto cut = [](int64_t n_tiles, int64_t range, int* splits, int* out) {
        *out = (int)std::min(std::max<int64_t>(range, 1), std::max<int64_t>(n_tiles, 1));
        *splits = (int)((n_tiles + *out - 1) / *out);
    };
    a->o_tiles = (int)(((int64_t)a->max_q * a->group + job_rows - 1) / job_rows);
    const int64_t o_jobs = (int64_t)a->batch * a->o_tiles * hk, o_keys = tiles(a->max_own), p_keys = tiles(a->prefix_len);
    const bool wide = type == TMAC_TYPE_F32;
    a->alone = o_keys + p_keys <= (wide ? kAloneTiles32 : p_keys ? kAloneTiles16 : kOwnTiles16) &&
               (!p_keys || o_jobs <= (int64_t)sms * jobs_of_sm(type, dim) ||
                p_keys * (wide ? kAloneRows32 : kAloneRows16) <= (int64_t)a->max_q * a->group);
    if (a->alone) {
        a->p_tiles = a->p_splits = a->p_range = 0;
        a->o_splits = 1;
        a->o_range = (int)std::max<int64_t>(1, o_keys + p_keys);
    } else {
        const int64_t rows = (int64_t)a->tokens * a->group;
        a->tc = type != TMAC_TYPE_F32 && rows >= kTcRowsLeast && rows * hk * a->prefix_len >= (dim == 64 ? kTcWork64 : kTcWork128) &&
                a->cache.page_shift >= 3;
        const int p_rows = a->tc ? kTcRows : job_rows;
        a->p_tiles = (int)((rows + p_rows - 1) / p_rows);
        const int64_t p_jobs = (int64_t)a->p_tiles * hk, room = (int64_t)sms * jobs_of_sm(type, dim) * (type == TMAC_TYPE_F32 ? 5 : 2) / 2;
        const int64_t p_work = p_jobs * p_keys, o_work = o_jobs * o_keys * 3 / 4;
        if (a->tc) {
            cut(p_keys, std::max<int64_t>(kTcRange, (p_work + 2 * sms - 1) / (2 * sms)), &a->p_splits, &a->p_range);
            cut(o_keys, (o_work + room - 1) / room, &a->o_splits, &a->o_range);
        } else {
            const int64_t range = (p_work + o_work + room - 1) / room;
            cut(p_keys, range, &a->p_splits, &a->p_range);
            cut(o_keys, range, &a->o_splits, &a->o_range);
        }
    }
    a->p_jobs = (int64_t)a->p_tiles * hk * a->p_splits;
    a->parts = a->p_splits + a->o_splits;
    return TMAC_OK;
}

size_t workspace_bytes_of(const AttnArgs& a)
{
    if (a.parts == 1) return 0;
    const size_t rows = (size_t)a.tokens * a.heads * a.parts;
    return rows * (size_t)a.cache.dim * sizeof(float) + rows * sizeof(float2);
}

template <typename T, int D>
int launch_attention(const AttnArgs& a, cudaStream_t s)
{
    const int64_t o_jobs = (int64_t)a.batch * a.o_tiles * a.cache.kv_heads * a.o_splits;
    if (a.p_jobs + o_jobs > 0x7FFFFFFF) return fail(TMAC_ERR_SHAPE, "too many jobs for one grid");
    AttnArgs rest = a;  // without the prefix's jobs, where the tcgen05 kernel takes them
    if (a.tc) {  // 16-bit elements
        const int rc = launch_prefix_tc(a, std::is_same_v<T, __half> ? TMAC_TYPE_F16 : TMAC_TYPE_BF16, s);
        if (rc) return rc;
        rest.p_jobs = 0;
    }
    const int64_t jobs = rest.p_jobs + o_jobs;
    if (jobs) {
        constexpr size_t smem = sizeof(MmaSmem<T, D>);
        auto fn = attn_mma_kernel<T, D>;
        static std::atomic<uint64_t> done{0};
        const int rc = set_once(done, a.device, [&] {
            return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        });
        if (rc) return rc;
        if (a.tc) {  // beside the prefix's jobs
            PdlScope beside;
            TMAC_CUDA_TRY(launch_k(fn, dim3((unsigned)jobs), dim3(kThreads), smem, s, rest));
        } else {
            fn<<<(unsigned)jobs, kThreads, smem, s>>>(rest);
            TMAC_CUDA_TRY(cudaGetLastError());
        }
    }
    if (a.parts == 1) return TMAC_OK;
    PdlScope overlap;  // the join's start overlaps the jobs' end; it waits for them before it reads
    TMAC_CUDA_TRY(launch_k(attn_join_kernel<T, D>, dim3((unsigned)(a.tokens * a.heads)), dim3(kThreads), 0, s, a));
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
    return plan(a, cache->type, num_sms(cache->device));
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

extern "C" int tmac_prefix_attention_engine(const tmac_paged_cache* cache, int heads, int tokens, int batch, int max_q,
                                            int prefix_len, int max_own)
{
    AttnArgs a = {};
    const int rc = prepare(cache, heads, tokens, batch, max_q, prefix_len, max_own, 0x7FFFFFFF, &a);
    return rc ? rc : a.p_jobs == 0 ? 0 : a.tc ? 2 : 1;
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
    if (!std::isfinite(scale)) return fail(TMAC_ERR_INVALID, "scale must be finite");
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
    a.device = cache->device;
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
