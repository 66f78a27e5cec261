// prefix_attention_tc.cu -- the shared prefix's part of prefix_attention on the
// 5th-generation tensor cores, for 16-bit elements and many query rows.
//
// A job is 128 rows (token, head of a key/value head's group) against a range of
// key tiles of 64.  Scores S = Q K^T are one tcgen05.mma chain per tile, both
// operands in shared memory; four softmax warps (a thread per row) read S from
// TMEM, keep the running maximum and sum, and store the weights P as 16-bit
// pairs into TMEM, where they are the first operand of O += P V; V's tile is the
// second as it lies ([keys][dims], the dims contiguous).  A row's scores are in its
// thread's registers before their weights are formed, so the next tile's product
// runs beneath them; P has two buffers.  O stays in TMEM.
//
// A weight is 2^(s - m) with m from the largest score of the row's first tile (in f16
// 8 less: its 11 bits end at 2^-14, and so at 2^-22 of the tile's largest weight), kept
// as long as no tile's sum of weights passes a limit (2^15 in f16, which ends at 2^16;
// 2^30 in bf16): a product and a rounding do not lose precision by a common factor.
// Only a tile that passes it pays for a new maximum, the rescaling of O, and its
// weights anew.  One thread issues the products, one warp the TMA copies of the pages
// (a box per page, 128-byte swizzle).
//
// Floor of the tile loop: the exponentials, 128 x 64 per tile at 16 a clock, 512 clocks
// against 256 of products at 64 dims.  Two CTAs share an SM: one's waits are the other's
// work.  896 rows a key/value head (two of 64 dims) over 32768 keys take 36.7 us with
// the join, 410 TFLOP/s: 24.3 us for every 32768 keys (950 clocks a tile on an SM), and
// 12.4 us whatever the length (2048 keys take 14.5), which are the launches, each CTA's
// start up to its first scores, its parts' way out and the join; no measurement tells
// these apart.  Three or four CTAs an SM, with the weights in the scores' place, take
// as long.
#include "prefix_attention.cuh"
#include "tcgen05.cuh"

namespace tmac {
namespace {

constexpr int kTcThreads = 6 * 32;  // warp 0 copies, warp 1 products, warps 2-5 softmax
constexpr int kSlab = kTile * 128;   // bytes of a tile's keys (or values) in 64 dims
constexpr int kQSlab = kTcRows * 128;
constexpr uint32_t kTmemCols = 256, kPCol = 64, kOCol = 128;  // S at 0, two buffers of P, O

template <int D>
struct Conf {
    static constexpr int kSlabs = D / 64, kStages = D == 64 ? 4 : 2;
    static constexpr int kBytes = kSlabs * kSlab, kQBytes = kSlabs * kQSlab;
    static constexpr size_t kSmem = 1024 + (size_t)kQBytes + 2 * kStages * kBytes + 256;
};
struct Bars {
    uint64_t q_full, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full, s_empty, p_full[2], pv_done[2], drain;
    uint32_t tmem;
    int failed;
};

// Second operand of O += P V: dims contiguous, 64-dim slabs of [keys][128 bytes]
// with the 128-byte swizzle; 8 keys (1024 bytes) apart along the product's depth.
TMAC_DEV uint64_t desc_v(uint32_t saddr)
{
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(kSlab >> 4) << 16;  // leading: the next 64 dims
    d |= (uint64_t)(1024 >> 4) << 32;   // stride: the next 8 keys
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// kind::f16, 32-bit sums, both operands f16 (0) or bf16 (1), 128 x n; v_dims: the
// second operand lies with its n contiguous.
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t bf16, uint32_t n, uint32_t v_dims)
{
    return (1u << 4) | (bf16 << 7) | (bf16 << 10) | (v_dims << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
TMAC_DEV void mma_f16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u));
}
TMAC_DEV void mma_f16_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u));
}
#define TMAC_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define TMAC_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
#define TMAC_I8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
TMAC_DEV void tmem_ld32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : TMAC_R8(r, 0), TMAC_R8(r, 8), TMAC_R8(r, 16), TMAC_R8(r, 24)
        : "r"(addr));
}
// Waits for this thread's loads; their registers pass through, so no use moves before it.
TMAC_DEV void tmem_wait_ld32(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : TMAC_RW8(r, 0), TMAC_RW8(r, 8), TMAC_RW8(r, 16), TMAC_RW8(r, 24)
                 :
                 : "memory");
}
TMAC_DEV void tmem_st32(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::TMAC_I8(r, 0),
        TMAC_I8(r, 8), TMAC_I8(r, 16), TMAC_I8(r, 24), "r"(addr)
        : "memory");
}
TMAC_DEV void tmem_st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::TMAC_I8(r, 0),
        TMAC_I8(r, 8), "r"(addr)
        : "memory");
}
TMAC_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two 32-bit floats at once.
struct Two {
    uint64_t v;
    TMAC_DEV Two(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
    TMAC_DEV explicit Two(uint64_t x) : v(x) {}
    TMAC_DEV void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
TMAC_DEV Two fma2(Two a, Two b, Two c)
{
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a.v), "l"(b.v), "l"(c.v));
    return Two(d);
}
TMAC_DEV Two add2(Two a, Two b)
{
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a.v), "l"(b.v));
    return Two(d);
}
// The weights 2^(x scale - m) of 32 scores, as pairs.  Returns their sum.
template <typename T>
TMAC_DEV float weights(const uint32_t (&x)[32], Two scale, Two base, uint32_t (&p)[16])
{
    Two sum[2] = {Two(0.0f, 0.0f), Two(0.0f, 0.0f)};
#pragma unroll
    for (int i = 0; i < 16; i++) {
        float e0, e1;
        fma2(Two(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale, base).get(e0, e1);
        const float p0 = exp2_fast(e0), p1 = exp2_fast(e1);
        sum[i & 1] = add2(sum[i & 1], Two(p0, p1));
        p[i] = pack2<T>(p0, p1);
    }
    float s0, s1;
    add2(sum[0], sum[1]).get(s0, s1);
    return __fadd_rn(s0, s1);
}

// Writes the warp's 32 rows of sums, as they lie in `rows` (kPad floats apart), each
// row's adjoining values by adjoining threads: the parts, or the rounded quotients
// when there are no others.
template <int D>
constexpr int kPad = D + 4;
template <typename T, int D>
TMAC_DEV void put_rows(const AttnArgs& a, const Job& j, const RowOf& row, bool mine, float l, const float* rows)
{
    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;
    const int lane = threadIdx.x & 31, c = lane % kLanes * 4;
    const int64_t at = a.parts == 1 ? row.token * a.out_stride + row.head * D
                                    : (((int64_t)row.token * a.heads + row.head) * a.parts + j.part) * D;
    const bool aligned = (((uintptr_t)a.out / sizeof(T)) | a.out_stride) % 4 == 0;
    for (int i = 0; i < 32; i += kAtOnce) {
        const int r = i + lane / kLanes;
        const int64_t to = __shfl_sync(0xffffffffu, at, r);
        const float sum = __shfl_sync(0xffffffffu, l, r);
        const bool wanted = __shfl_sync(0xffffffffu, (int)mine, r);
        float4 x = *reinterpret_cast<const float4*>(rows + r * kPad<D> + c);
        if (!wanted) continue;
        if (sum == 0.0f) x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // saw no key
        if (a.parts > 1) {
            *reinterpret_cast<float4*>(a.part_o + to + c) = x;
            continue;
        }
        const float by = sum == 0.0f ? 0.0f : __frcp_rn(sum);
        T* out = (T*)a.out + to + c;
        const uint2 y = make_uint2(pack2<T>(__fmul_rn(x.x, by), __fmul_rn(x.y, by)), pack2<T>(__fmul_rn(x.z, by), __fmul_rn(x.w, by)));
        if (aligned) {
            *reinterpret_cast<uint2*>(out) = y;
        } else {
            const T* e = reinterpret_cast<const T*>(&y);
#pragma unroll
            for (int k = 0; k < 4; k++) out[k] = e[k];
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTcThreads, 2)
    attn_tc_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map)
{
    using C = Conf<D>;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + (1024 - (smem_addr(smem_raw) & 1023)) % 1024;
    uint8_t *q_s = smem, *k_s = q_s + C::kQBytes, *v_s = k_s + C::kStages * C::kBytes;
    Bars& bar = *reinterpret_cast<Bars*>(v_s + C::kStages * C::kBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch();  // the own part may start beside this kernel
    Job j;
    find_job<kTcRows>(a, &j);
    const int key0 = j.tile0 * kTile, key1 = min(j.p_keys, j.tile1 * kTile);
    const int n_tiles = tiles_of(key1 - key0);

    // the softmax threads' rows of Q, on their way while the rest is set up
    const int quarter = warp & 3, r = quarter * 32 + lane;
    RowOf row = {0, 0, 0x7FFFFFFF, 0};
    uint4 q[D / 8];
    if (warp >= 2) {
        if (r < j.rows) row = find_row(a, j, r);
        const T* src = (const T*)a.q + row.token * a.q_stride + row.head * D;
        const bool aligned = ((uintptr_t)a.q | (uintptr_t)(a.q_stride * sizeof(T))) % 16 == 0;
#pragma unroll
        for (int c = 0; c < D / 8; c++) {
            q[c] = make_uint4(0, 0, 0, 0);
            if (r >= j.rows) continue;
            if (aligned) {
                q[c] = __ldg(reinterpret_cast<const uint4*>(src) + c);
            } else {
                T e[8];
#pragma unroll
                for (int i = 0; i < 8; i++) e[i] = src[8 * c + i];
                q[c] = *reinterpret_cast<const uint4*>(e);
            }
        }
    }

    if (threadIdx.x == 0) {
        mbar_init(&bar.q_full, 128);
        for (int i = 0; i < C::kStages; i++) {
            mbar_init(&bar.k_full[i], 1);
            mbar_init(&bar.k_empty[i], 1);
            mbar_init(&bar.v_full[i], 1);
            mbar_init(&bar.v_empty[i], 1);
        }
        mbar_init(&bar.s_full, 1);
        mbar_init(&bar.s_empty, 128);
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar.p_full[i], 128);
            mbar_init(&bar.pv_done[i], 1);
        }
        mbar_init(&bar.drain, 1);
        bar.failed = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&bar.tmem, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem;
    // The use-th completion (from 0) of a barrier.  By parity: at the time of the wait the
    // barrier must have seen use or use + 1 of them, which is why some come in pairs.
    const auto wait = [&](uint64_t* b, int use) {
        if (mbar_wait_bounded(b, (uint32_t)(use & 1), a.err)) return true;
        *(volatile int*)&bar.failed = 1;
        return false;
    };

    if (warp == 0) {
        // ---- copies: a lane to a page
        const int shift = a.cache.page_shift, page_rows = min(1 << shift, kTile), boxes = kTile / page_rows;
        const int rows_all = (int)((a.cache.n_pages * a.cache.kv_heads) << shift);  // past the pool: reads zeros
        int issued = 0;
        bool ok = true;
        for (int t = 0; t < n_tiles; t++) {
            const int st = t % C::kStages, key = key0 + t * kTile;
            const int here = min(boxes, (key1 - key + page_rows - 1) / page_rows);
            int row = rows_all;
            if (lane < here) {
                const int g = key + lane * page_rows;
                const int64_t page = a.prefix_pages[g >> shift];
                if (page >= 0 && page < a.cache.n_pages)
                    row = (int)((page * a.cache.kv_heads + j.kvh) << shift) + (g & ((1 << shift) - 1));
                else
                    record_error(a.err, TMAC_ERR_BOUNDS);
            }
            const auto copy = [&](uint64_t* full, uint64_t* empty, uint8_t* to, const CUtensorMap* map) {
                if (ok && t >= C::kStages) ok = wait(empty, t / C::kStages - 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(here * page_rows * 128 * C::kSlabs));
                __syncwarp();
                if (lane < here)
                    for (int h = 0; h < C::kSlabs; h++) tma_load_2d(to + h * kSlab + lane * page_rows * 128, map, h * 64, row, full);
            };
            copy(&bar.k_full[st], &bar.k_empty[st], k_s + st * C::kBytes, &k_map);
            if (!ok) break;
            issued = 2 * t + 1;
            copy(&bar.v_full[st], &bar.v_empty[st], v_s + st * C::kBytes, &v_map);
            if (!ok) break;
            issued = 2 * t + 2;
        }
        if (*(volatile int*)&bar.failed)  // wait for the copies in flight, within the limit again
            for (int i = max(0, issued - 2 * C::kStages); i < issued; i++)
                mbar_wait_bounded(i & 1 ? &bar.v_full[i / 2 % C::kStages] : &bar.k_full[i / 2 % C::kStages],
                                  (uint32_t)(i / 2 / C::kStages & 1), a.err);
    } else if (warp == 1) {
        // ---- products
        if (lane == 0) {
            constexpr uint32_t kBf16 = std::is_same_v<T, __nv_bfloat16>;
            constexpr uint32_t kIdS = idesc_f16(kBf16, kTile, 0), kIdO = idesc_f16(kBf16, D, 1);
            bool ok = wait(&bar.q_full, 0);
            const auto scores = [&](int t) {
                const int st = t % C::kStages;
                if (!ok || !(ok = wait(&bar.k_full[st], t / C::kStages))) return;
                if (t >= 1 && !(ok = wait(&bar.s_empty, t - 1))) return;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < D / 16; i++)
                    mma_f16(tmem, desc_sw128(smem_addr(q_s) + i / 4 * kQSlab + i % 4 * 32),
                            desc_sw128(smem_addr(k_s + st * C::kBytes) + i / 4 * kSlab + i % 4 * 32), kIdS, i > 0);
                mma_commit(&bar.k_empty[st]);
                mma_commit(&bar.s_full);
            };
            scores(0);
            for (int t = 0; ok && t < n_tiles; t++) {
                if (t + 1 < n_tiles) scores(t + 1);
                const int st = t % C::kStages;
                if (!ok || !(ok = wait(&bar.v_full[st], t / C::kStages)) || !(ok = wait(&bar.p_full[t % 2], t / 2))) break;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < kTile / 16; i++)
                    mma_f16_tmem(tmem + kOCol, tmem + kPCol + t % 2 * 32 + 8 * i, desc_v(smem_addr(v_s + st * C::kBytes) + i * 16 * 128),
                                 kIdO, t > 0 || i > 0);
                mma_commit(&bar.v_empty[st]);
                mma_commit(&bar.pv_done[t % 2]);
            }
            mma_commit(&bar.drain);
            mbar_wait_bounded(&bar.drain, 0, a.err);  // nothing in flight when TMEM is freed
        }
        __syncwarp();
    } else {
        // ---- softmax: thread = row
        const uint32_t mine = tmem + ((uint32_t)quarter << 21);  // lane quarter * 32 of TMEM
        const bool idle = quarter * 32 >= j.rows;  // no row of this warp: its weights are not read
        {
            // a negative scale turns Q's signs, so that the largest score has the largest weight
            const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0;
#pragma unroll
            for (int c = 0; c < D / 8; c++)
                *reinterpret_cast<uint4*>(q_s + c / 8 * kQSlab + r * 128 + ((c & 7) ^ (r & 7)) * 16) =
                    make_uint4(q[c].x ^ sign, q[c].y ^ sign, q[c].z ^ sign, q[c].w ^ sign);
            fence_proxy_async_smem();
            mbar_arrive(&bar.q_full);
        }
        // exponentials are powers of 2; not 0, so that a masked score's -inf stays one
        const float scale = fmaxf(__fmul_rn(fabsf(a.scale), 1.44269504f), 1e-37f);
        constexpr float kLimit = std::is_same_v<T, __half> ? 32768.0f : 1073741824.0f;
        constexpr float kFirstPower = std::is_same_v<T, __half> ? 8.0f : 0.0f;  // the largest weight under a new m
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        // V's rows past the keys hold what the page or an earlier tile holds: zeros instead
        const auto zero_values = [&](int t) {
            const int st = t % C::kStages;
            if (!__all_sync(0xffffffffu, wait(&bar.v_full[st], t / C::kStages))) return false;
            if (r < kTile && r >= key1 - (key0 + t * kTile))
                for (int h = 0; h < C::kSlabs; h++)
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        *reinterpret_cast<uint4*>(v_s + st * C::kBytes + h * kSlab + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            return true;
        };
        for (int t = 0; t < n_tiles; t++) {
            const int key = key0 + t * kTile, seen = min(row.p_limit, key1) - key;
            if (!(ok = __all_sync(0xffffffffu, wait(&bar.s_full, t)))) break;
            tc_fence_after();
            if (idle) {
                mbar_arrive(&bar.s_empty);
                if (t > 1 && !(ok = __all_sync(0xffffffffu, wait(&bar.pv_done[t % 2], t / 2 - 1)))) break;
            } else {
                uint32_t x[2][32], p[2][16];
                tmem_ld32(mine, x[0]);
                tmem_ld32(mine + 32, x[1]);
                tmem_wait_ld32(x[0]);
                tmem_wait_ld32(x[1]);
                tc_fence_before();
                mbar_arrive(&bar.s_empty);
                if (__any_sync(0xffffffffu, seen < kTile)) {
#pragma unroll
                    for (int c = 0; c < 64; c++)
                        if (c >= seen) x[c / 32][c % 32] = 0xFF800000u;  // -inf
                }
                // this buffer's last weights have been read
                if (t > 1 && !(ok = __all_sync(0xffffffffu, wait(&bar.pv_done[t % 2], t / 2 - 1)))) break;
                float sum = 0.0f;
                for (bool fits = m > -INFINITY, found = false;; found = true) {
                    if (__any_sync(0xffffffffu, !fits)) {  // a larger m
                        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 64; c++) top[c & 3] = fmaxf(top[c & 3], __fmul_rn(__uint_as_float(x[c / 32][c % 32]), scale));
                        const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                        const float mx = fits ? m : fmaxf(m, __fsub_rn(most, kFirstPower));
                        const float al = mx == m ? 1.0f : exp2_fast(__fsub_rn(m, mx));
                        m = mx;
                        l = __fmul_rn(l, al);
                        if (t > 0) {  // the sums so far must be complete
                            if (!(ok = __all_sync(0xffffffffu, wait(&bar.pv_done[(t - 1) % 2], (t - 1) / 2)))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D / 32; c++) {
                                uint32_t y[32];
                                tmem_ld32(mine + kOCol + 32 * c, y);
                                tmem_wait_ld32(y);
#pragma unroll
                                for (int i = 0; i < 32; i++) y[i] = __float_as_uint(__fmul_rn(__uint_as_float(y[i]), al));
                                tmem_st32(mine + kOCol + 32 * c, y);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.0f : -m;
                    const Two scale2(scale, scale), base2(base, base);
                    sum = __fadd_rn(weights<T>(x[0], scale2, base2, p[0]), weights<T>(x[1], scale2, base2, p[1]));
                    fits = !(sum > kLimit);
                    if (found || __all_sync(0xffffffffu, fits)) break;
                }
                if (!ok) break;
                tmem_st16(mine + kPCol + t % 2 * 32, p[0]);
                tmem_st16(mine + kPCol + t % 2 * 32 + 16, p[1]);
                l = __fadd_rn(l, sum);
            }
            if (key1 - key < kTile && !(ok = zero_values(t))) break;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&bar.p_full[t % 2]);
        }
        for (int t = max(0, n_tiles - 2); ok && t < n_tiles; t++) ok = __all_sync(0xffffffffu, wait(&bar.pv_done[t % 2], t / 2));
        if (ok && !idle) {
            tc_fence_after();
            bool finite = true;
            // the tiles' place is free: every product has run
            float* rows = reinterpret_cast<float*>(smem) + quarter * 32 * kPad<D>;
            static_assert(4 * 32 * kPad<D> * sizeof(float) <= C::kQBytes + 2 * C::kStages * C::kBytes, "room for the rows");
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                uint32_t x[32];
                tmem_ld32(mine + kOCol + 32 * c, x);
                tmem_wait_ld32(x);
#pragma unroll
                for (int i = 0; i < 32; i++) finite &= fabsf(__uint_as_float(x[i])) < INFINITY;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    *reinterpret_cast<uint4*>(rows + lane * kPad<D> + 32 * c + 4 * i) =
                        make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            }
            __syncwarp();
            const bool wanted = r < j.rows && finite;
            if (wanted && a.parts > 1) a.part_ml[((int64_t)row.token * a.heads + row.head) * a.parts + j.part] = make_float2(m, l);
            put_rows<T, D>(a, j, row, wanted, l, rows);
            for (uint32_t again = __ballot_sync(0xffffffffu, r < j.rows && !finite); again; again &= again - 1)
                row_by_keys<T, D>(a, j, quarter * 32 + __ffs(again) - 1);
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tmem, kTmemCols);
    if (a.q_start && a.parts == 1) clear_rows<T, D, kTcRows>(a);
}

template <typename T, int D>
int launch_tc(const AttnArgs& a, cudaStream_t s)
{
    using C = Conf<D>;
    auto encode = encode_fn();
    if (!encode) return fail(TMAC_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    const int page_rows = std::min(1 << a.cache.page_shift, kTile);
    CUtensorMap maps[2];
    for (int i = 0; i < 2; i++) {
        const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)(a.cache.n_pages * a.cache.kv_heads) << a.cache.page_shift};
        const cuuint64_t strides[1] = {D * sizeof(T)};
        const cuuint32_t box[2] = {64, (cuuint32_t)page_rows}, elem[2] = {1, 1};
        const auto type = std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        if (encode(&maps[i], type, 2, i ? a.cache.v : a.cache.k, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return fail(TMAC_ERR_CUDA, "cuTensorMapEncodeTiled failed for the cache's pages");
    }
    static std::atomic<uint64_t> done{0};
    const int rc = set_once(done, a.device, [&] {
        return cudaFuncSetAttribute(attn_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem);
    });
    if (rc) return rc;
    attn_tc_kernel<T, D><<<(unsigned)a.p_jobs, kTcThreads, C::kSmem, s>>>(a, maps[0], maps[1]);
    TMAC_CUDA_TRY(cudaGetLastError());
    return TMAC_OK;
}

}  // namespace

int launch_prefix_tc(const AttnArgs& a, int type, cudaStream_t s)
{
    if (type == TMAC_TYPE_F16) return a.cache.dim == 64 ? launch_tc<__half, 64>(a, s) : launch_tc<__half, 128>(a, s);
    return a.cache.dim == 64 ? launch_tc<__nv_bfloat16, 64>(a, s) : launch_tc<__nv_bfloat16, 128>(a, s);
}

}  // namespace tmac
