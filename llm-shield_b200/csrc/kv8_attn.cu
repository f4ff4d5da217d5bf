// kv8_attn.cu — grouped-query attention over the 8-bit paged cache (jv_kv8_attention).
//
// o = sum_j softmax_j(scale q . k_j) v_j with k_j = ks(j) kint_j and v_j = vs(j) vint_j, where ks and vs
// are the scales of key j's block of 16. The scales never touch the matrices: with
//   e_j = scale ks(j) (q . kint_j) + log2 vs(j)   (in log2 units),   w_j = 2^(e_j - M),   M >= max e_j - 8
// the output is  sum_j w_j vint_j / sum_j (w_j / vs(j)),  so the products run on exact integers (an
// int8 is exact in fp16), w_j <= 2^8 is the only rounded operand (fp16: half a step, 2^-11 of a weight above
// 2^-14 and 2^-25 below), and sums, M and the softmax denominator are fp32. A block whose values are all zero
// has vs = PG_ZERO_SCALE. bf16 queries are taken to fp16 by a power of two per row.
//
// Here: the requests of few query rows, whose time is the cache's bytes. (kv8_attn_tc.cu has the others.)
// The products are mma.sync m16n8k16 with the keys on the 16-row side and the query rows (new token x
// head of the group) on the 8-column side: S^T = K Q^T, O^T = V^T P^T. The order of the 128
// dimensions inside a product is free, so a lane loads 16 consecutive int8 of its rows straight from
// the cache's rows into fragments; S^T becomes the operand P^T by one movmatrix per 8 x 8 block.
#include <atomic>
#include <cmath>
#include <string>

#include <cuda.h>
#include <cuda_bf16.h>

#include "paged.h"
#include "tc_common.cuh"

namespace jv {
namespace {

constexpr float KA_LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float lg2f(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// Two bytes (biased by 128) of x as an fp16 pair of the int8 they stand for: 0x64bb is 1024 + bb.
__device__ __forceinline__ uint32_t pair_f16(uint32_t x, uint32_t sel) {
    const uint32_t w = __byte_perm(x, 0x64646464u, sel);
    const __half2 h = __hsub2(*(const __half2*)&w, __floats2half2_rn(1152.f, 1152.f));
    return *(const uint32_t*)&h;
}

__device__ __forceinline__ float2 unpack_bf16(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&h;
}

// A row of 128 bf16 held by the four lanes of a group (16 pairs each), as fp16 times the power of two that is
// returned: the one that puts the row's largest magnitude in [2^13, 2^14). Exact but for values 2^27 below it.
__device__ __forceinline__ float q_to_f16(uint32_t (&q)[16]) {
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float2 x = unpack_bf16(q[e]);
        amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int ex = min(max((int)((__float_as_uint(amax) >> 23) & 0xff), 14), 254);  // 2^(ex - 127) <= amax
    const float up = __uint_as_float((uint32_t)(267 - ex) << 23);                     // 2^(13 - (ex - 127))
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float2 x = unpack_bf16(q[e]);
        q[e] = pack2<__half>(x.x * up, x.y * up);
    }
    return up;
}

// Stores four outputs of a row; true where fp16 does not hold one.
template <class T>
__device__ __forceinline__ bool store_row(const AttnKArgs& a, int start, int kvh, int row, int d4, float4 o, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // no visible key: zeros (a NaN stays one)
    T* dst = (T*)a.q.out + (int64_t)(start + row / a.b.group) * a.q.out_token +
             (int64_t)(kvh * a.b.group + row % a.b.group) * a.q.out_head + 4 * d4;
    o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
    *(uint2*)dst = make_uint2(pack2<T>(o.x, o.y), pack2<T>(o.z, o.w));
    return outside<T>(o);
}

// ------------------------------------------------------------ small requests

// Small requests: persistent warps, each on its own, over (chunk of a request, row tile, KV head). A warp
// streams its keys through two stages of 32 (K and V, one TMA tile each, stored with the 128-byte swizzle so
// that the fragment loads below meet no bank twice); it refills a stage as soon as it has used it, with its
// next keys or already with the first of its next item. Nothing joins the warps: a chunk's result goes to
// the workspace (k_kv8_join), or out when the request has one chunk. Bound by HBM: 12 warps keep 96 KB per SM
// in flight; a 16-key tile costs about 360 instructions (64 requests of 300 to 8000 keys: 98 us, 5.5 TB/s).
// With two 8-row tiles per warp (NT = 2) the registers leave 8 warps per SM, with a third stage each, and latency
// is what bounds it (24 requests of 2 to 6 new tokens: 82 us; query fragments in shared memory, for 12 warps: 108;
// three 8-row tiles: 92).
constexpr int KS_WARPS = 4;
template <int NT>
struct Ks {
    static constexpr int keys = 32;                 // per stage
    static constexpr int ctas = NT == 1 ? 3 : 2;    // per SM
    static constexpr int stages = NT == 1 ? 2 : 3;
    static constexpr int half = keys * PG_DIM;      // bytes of K or V in a stage
    static constexpr int ring = stages * 2 * half;  // bytes of a warp's stages
    static constexpr int smem = KS_WARPS * ring + 1024;
};
// A place in a warp's ring and the parity of its current use.
template <int STAGES>
struct Turn {
    uint32_t stage = 0, parity = 0;
    __device__ __forceinline__ void next() {
        if (++stage == STAGES) stage = 0, parity ^= 1;
    }
};

__device__ __forceinline__ void tma_keys(uint32_t dst, const CUtensorMap* map, int row, int kvh, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(
            dst),
        "l"(map), "r"(0), "r"(row), "r"(kvh), "r"(page), "r"(bar)
        : "memory");
}

// One work item of a warp: its rows and keys; lane j holds page `page0 + j` of the request.
struct KsItem {
    int start, n_new, len, row0, n_rows, kvh, item, chunks, lo, hi, page0, pages;
    bool valid;
};

template <class T, int NT>
__global__ void __launch_bounds__(KS_WARPS * 32, Ks<NT>::ctas) k_kv8_small(AttnKArgs a, const __grid_constant__ CUtensorMap map) {
    constexpr int KEYS = Ks<NT>::keys, HALF = Ks<NT>::half, STAGES = Ks<NT>::stages, H = KEYS / PG_BLOCK;
    extern __shared__ uint8_t ks_raw[];
    __shared__ uint64_t bars[KS_WARPS * STAGES];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, i = lane & 3;
    uint8_t* sm = ks_raw + ((1024u - (s_addr(ks_raw) & 1023u)) & 1023u) + warp * Ks<NT>::ring;
    const uint32_t base = s_addr(sm), full = s_addr(bars + warp * STAGES);
    if (lane == 0) {
        for (int s = 0; s < STAGES; s++) mbar_init(full + 8 * s, 1);
        fence_barrier_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();  // after the wait: what the plan wrote is then complete for the kernel after this one too
    const int kvh_n = a.c.kv_heads, group = a.b.group;
    const int64_t total = (int64_t)min((int64_t)max(a.v.head[0], 0), a.v.small_cap) * kvh_n;
    const int64_t stride = (int64_t)gridDim.x * KS_WARPS;
    int64_t unit = (int64_t)blockIdx.x * KS_WARPS + warp;

    auto fetch = [&](int64_t u, int4& x, int4& y) {
        if (u < total) {
            x = a.v.small_items[2 * (u / kvh_n)];
            y = a.v.small_items[2 * (u / kvh_n) + 1];
        } else {
            x = make_int4(-1, 0, 0, 0);
            y = make_int4(0, 0, 0, 0);
        }
    };
    auto decode = [&](int64_t u, int4 x, int4 y) {
        KsItem t;
        t.item = (int)(u / kvh_n), t.kvh = (int)(u % kvh_n);
        t.start = y.x, t.n_new = y.y, t.len = y.z, t.chunks = x.z;
        t.row0 = x.w * PG_ROW_TILE;
        t.valid = x.x >= 0 && x.x < a.b.requests && rows_in_bounds(a.b, t.start, t.n_new, t.len) && t.row0 >= 0 &&
                  t.row0 < t.n_new * group && x.y >= 0 && x.z >= 1;
        if (!t.valid) t.n_new = t.len = t.row0 = 0;
        t.n_rows = min(min(t.n_new * group - t.row0, a.rows), 8 * NT);
        const int ck = pg_chunk_keys(t.len, t.n_new * group);
        const int64_t from = (int64_t)x.y * ck;
        t.lo = (int)min(from, (int64_t)t.len);
        t.hi = (int)min(from + ck, (int64_t)t.len);
        if (a.window > 0) t.lo = max(t.lo, t.len - t.n_new + t.row0 / group + 1 - a.window);
        if (!t.valid || t.lo >= t.hi) t.lo = t.hi = 0;
        t.page0 = t.lo / PG_TOKENS;
        t.pages = t.page0 * PG_TOKENS + lane * PG_TOKENS < t.hi ? a.b.block_table[(int64_t)x.x * a.b.max_blocks + t.page0 + lane] : 0;
        return t;
    };
    // The stage of `turn` takes step t of an item (keys KEYS t ..); a page that is not in the cache is not read.
    auto issue = [&](const KsItem& it, int t, Turn<STAGES>& turn) {
        const int page = __shfl_sync(0xffffffffu, it.pages, t * KEYS / PG_TOKENS - it.page0);
        const bool there = (unsigned)page < (unsigned)a.c.pages;
        if (lane == 0) {
            const uint32_t bar = full + 8 * turn.stage, dst = base + turn.stage * 2 * HALF;
            mbar_expect_tx(bar, there ? 2 * HALF : 0);
            if (there) {
                const int row = t * KEYS % PG_TOKENS;
                tma_keys(dst, &map, row, it.kvh, page, bar);
                tma_keys(dst + HALF, &map, PG_TOKENS + row, it.kvh, page, bar);
            } else {
                paged_report(a.b.status, JV_ERR_RANGE, PS_ATTN_PAGE);
            }
        }
        __syncwarp();
        turn.next();
    };
    auto scales_of = [&](const KsItem& it, int t, float (&k)[H], float (&v)[H]) {
        const int page = __shfl_sync(0xffffffffu, it.pages, t * KEYS / PG_TOKENS - it.page0);
        const bool there = (unsigned)page < (unsigned)a.c.pages;
        if (there) {
            const float* p = a.c.scales + (int64_t)page * a.c.scale_stride + it.kvh * 8 + t * KEYS % PG_TOKENS / PG_BLOCK;
#pragma unroll
            for (int h = 0; h < H; h++) k[h] = p[h], v[h] = p[4 + h];
        }
        return there;
    };

    // Rows of a 16-key tile by fragment row: evens stay, odds are exchanged 4 apart, so that the lanes that load
    // together (two fragment rows of K, four key pairs of V) find their 16-byte chunks in eight different places.
    const int krow = (g & 1) ? ((g - 1) ^ 4) + 1 : g;
    const int vrow = (2 * i ^ 4) + 1;
    const uint32_t k_off = krow * PG_DIM, k_c0 = (i ^ (krow & 7)) << 4, k_c1 = ((4 + i) ^ (krow & 7)) << 4;
    const uint32_t v_off0 = 2 * i * PG_DIM + ((g ^ (2 * i)) << 4), v_off1 = vrow * PG_DIM + ((g ^ vrow) << 4);

    int4 px, py;
    fetch(unit, px, py);
    KsItem cur = decode(unit, px, py);
    fetch(unit + stride, px, py);
    Turn<STAGES> in, out;     // stages filled and used
    int flight = 0;           // filled and not yet used
    int at = cur.lo / KEYS;   // next step of `cur` to issue
    for (; flight < STAGES && at * KEYS < cur.hi; flight++) issue(cur, at++, in);
    for (; unit < total; unit += stride) {
        const KsItem nxt = decode(unit + stride, px, py);
        fetch(unit + 2 * stride, px, py);
        int nat = nxt.lo / KEYS;
        if (cur.valid) {
            uint32_t qr[NT][16];
            float qs[NT][2], qb[NT][2], acc[NT][8][4], m[NT][2], l[NT][2];
            const int first = cur.len - cur.n_new + cur.row0 / group;
            const int last = cur.len - cur.n_new + (cur.row0 + cur.n_rows - 1) / group;
            const int all_hi = min(first + 1, cur.hi), all_lo = max(cur.lo, a.window > 0 ? last + 1 - a.window : 0);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const int row = 8 * n + g;
                uint32_t qf[16];
#pragma unroll
                for (int e = 0; e < 16; e++) qf[e] = 0;
                if (row < cur.n_rows) {
                    const int r = cur.row0 + row;
                    const T* src = (const T*)a.q.in + (int64_t)(cur.start + r / group) * a.q.in_token +
                                   (int64_t)(cur.kvh * group + r % group) * a.q.in_head + 16 * i;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint4 x = *(const uint4*)(src + 64 * (j >> 1) + 8 * (j & 1));
                        qf[4 * j] = x.x, qf[4 * j + 1] = x.y, qf[4 * j + 2] = x.z, qf[4 * j + 3] = x.w;
                    }
                }
                float f = 1.f;
                if (std::is_same<T, __nv_bfloat16>::value) f = 1.f / q_to_f16(qf);
                f *= a.scale;
                // The K fragments are the bytes b + 128 as fp16 subnormals, (b + 128) 2^-24: an exact operand for
                // one byte permute. q . kint = 2^24 (q . frag) - 128 sum q; the sum of the row is taken here.
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const float2 x = __half22float2(*(const __half2*)&qf[e]);
                    sum += x.x + x.y;
                }
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    qr[n][e] = qf[e];
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int col = 2 * i + e;
                    qs[n][e] = __shfl_sync(0xffffffffu, f, 4 * col);
                    qb[n][e] = -128.f * __shfl_sync(0xffffffffu, sum, 4 * col) * qs[n][e];
                    qs[n][e] *= 16777216.f;
                    m[n][e] = -INFINITY;
                    l[n][e] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[n][j][e] = 0.f;
            }
            float ks[H], vs[H];
            bool there = false;
            if (cur.lo < cur.hi) there = scales_of(cur, cur.lo / KEYS, ks, vs);
            for (int t = cur.lo / KEYS; t * KEYS < cur.hi; t++) {
                if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * out.stage, out.parity))) {
                    if (lane == 0) paged_report(a.b.status, JV_ERR_DEVICE_TIMEOUT, PS_ATTN_WAIT);
                    for (out.next(); --flight > 0; out.next()) mbar_wait(full + 8 * out.stage, out.parity);  // copies still in flight
                    return;
                }
                float ks_t[H], vs_t[H];
                const bool there_t = there;
                const int key0 = t * KEYS;
#pragma unroll
                for (int h = 0; h < H; h++) {
                    ks_t[h] = ks[h];
                    // a block of zeros, or one without a key of the request
                    vs_t[h] = vs[h] > 0.f && key0 + h * PG_BLOCK < cur.hi ? vs[h] : PG_ZERO_SCALE;
                }
                if ((t + 1) * KEYS < cur.hi) there = scales_of(cur, t + 1, ks, vs);
                if (there_t) {
                    const bool all = key0 >= all_lo && key0 + KEYS <= all_hi;
                    {
                        const uint8_t* kp = sm + out.stage * 2 * HALF;
                        float s[H][NT][4];
#pragma unroll
                        for (int h = 0; h < H; h++) {
                            uint4 kr[2][2];
#pragma unroll
                            for (int r = 0; r < 2; r++) {
                                kr[r][0] = *(const uint4*)(kp + h * PG_BLOCK * PG_DIM + 8 * r * PG_DIM + k_off + k_c0);
                                kr[r][1] = *(const uint4*)(kp + h * PG_BLOCK * PG_DIM + 8 * r * PG_DIM + k_off + k_c1);
                            }
#pragma unroll
                            for (int n = 0; n < NT; n++)
#pragma unroll
                                for (int e = 0; e < 4; e++) s[h][n][e] = 0.f;
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                const uint32_t w0[4] = {kr[0][j].x, kr[0][j].y, kr[0][j].z, kr[0][j].w};
                                const uint32_t w1[4] = {kr[1][j].x, kr[1][j].y, kr[1][j].z, kr[1][j].w};
#pragma unroll
                                for (int w = 0; w < 4; w++) {
                                    const uint32_t x0 = w0[w] ^ 0x80808080u, x1 = w1[w] ^ 0x80808080u;
                                    const uint32_t f[4] = {__byte_perm(x0, 0, 0x4140), __byte_perm(x1, 0, 0x4140),
                                                           __byte_perm(x0, 0, 0x4342), __byte_perm(x1, 0, 0x4342)};
#pragma unroll
                                    for (int n = 0; n < NT; n++) mma_f16(s[h][n], f, qr[n][8 * j + 2 * w], qr[n][8 * j + 2 * w + 1]);
                                }
                            }
                        }
                        uint32_t pb[H][NT][2];
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float e[H][4], mx[2], iv[H];
#pragma unroll
                            for (int h = 0; h < H; h++) {
                                const float kk = ks_t[h], lv = lg2f(vs_t[h]);
                                iv[h] = __frcp_rn(vs_t[h]);
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    const float ka = kk * qs[n][c], kb = fmaf(kk, qb[n][c], lv);
                                    e[h][c] = fmaf(s[h][n][c], ka, kb);
                                    e[h][c + 2] = fmaf(s[h][n][c + 2], ka, kb);
                                }
                            }
                            if (!all) {
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    const int r = 8 * n + 2 * i + c, pos = cur.len - cur.n_new + (cur.row0 + r) / group;
                                    const int hi_key = r < cur.n_rows ? min(pos + 1, cur.hi) : 0, lo_key = a.window > 0 ? pos + 1 - a.window : 0;
#pragma unroll
                                    for (int h = 0; h < H; h++)
#pragma unroll
                                        for (int x = c; x < 4; x += 2) {
                                            const int key = key0 + h * PG_BLOCK + krow + 8 * (x >> 1);
                                            if (key >= hi_key || key < lo_key) e[h][x] = -INFINITY;
                                        }
                                }
                            }
                            bool move = false;
#pragma unroll
                            for (int c = 0; c < 2; c++) {
                                mx[c] = fmaxf(e[0][c], e[0][c + 2]);
                                if (H == 2) mx[c] = fmaxf(mx[c], fmaxf(e[H - 1][c], e[H - 1][c + 2]));
                                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 4));
                                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 8));
                                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 16));
                                move |= mx[c] > m[n][c] + 8.f;
                            }
                            // the reference moves only when a score passes it by 2^8 (weights stay below 2^8)
                            if (__any_sync(0xffffffffu, move)) {
                                float alpha[2];
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    const float mn = fmaxf(m[n][c], mx[c]);
                                    alpha[c] = m[n][c] == -INFINITY ? 0.f : ex2(m[n][c] - mn);
                                    m[n][c] = mn;
                                    l[n][c] *= alpha[c];
                                }
#pragma unroll
                                for (int j = 0; j < 8; j++)
#pragma unroll
                                    for (int x = 0; x < 4; x++) acc[n][j][x] *= alpha[x & 1];
                            }
#pragma unroll
                            for (int h = 0; h < H; h++) {
#pragma unroll
                                for (int c = 0; c < 2; c++) {
                                    const float ref = m[n][c] == -INFINITY ? 0.f : m[n][c];
                                    e[h][c] = ex2(e[h][c] - ref);
                                    e[h][c + 2] = ex2(e[h][c + 2] - ref);
                                    l[n][c] = fmaf(e[h][c] + e[h][c + 2], iv[h], l[n][c]);
                                }
                                pb[h][n][0] = movmatrix_trans(pack2<__half>(e[h][0], e[h][1]));
                                pb[h][n][1] = movmatrix_trans(pack2<__half>(e[h][2], e[h][3]));
                            }
                        }
                        // O^T += V^T P^T: dimension 16 g + 2 j is the tile's row g, 16 g + 2 j + 1 its row g + 8. The
                        // V fragments are signed integers (1024 + b + 128 - 1152): sums over thousands of keys would
                        // lose what an offset left in them.
#pragma unroll
                        for (int h = 0; h < H; h++) {
                            const uint8_t* vp = kp + HALF + h * PG_BLOCK * PG_DIM;
                            const uint4 ra = *(const uint4*)(vp + v_off0), rb = *(const uint4*)(vp + v_off1);
                            const uint4 rc = *(const uint4*)(vp + v_off0 + 8 * PG_DIM), rd = *(const uint4*)(vp + v_off1 + 8 * PG_DIM);
                            const uint32_t va[4] = {ra.x, ra.y, ra.z, ra.w}, vb[4] = {rb.x, rb.y, rb.z, rb.w};
                            const uint32_t vc[4] = {rc.x, rc.y, rc.z, rc.w}, vd[4] = {rd.x, rd.y, rd.z, rd.w};
#pragma unroll
                            for (int w = 0; w < 4; w++)
#pragma unroll
                                for (int u = 0; u < 2; u++) {
                                    const uint32_t sel = u ? 0x7362 : 0x5140;
                                    const uint32_t lo = __byte_perm(va[w], vb[w], sel) ^ 0x80808080u;
                                    const uint32_t hi = __byte_perm(vc[w], vd[w], sel) ^ 0x80808080u;
                                    const uint32_t f[4] = {pair_f16(lo, 0x4140), pair_f16(lo, 0x4342), pair_f16(hi, 0x4140), pair_f16(hi, 0x4342)};
#pragma unroll
                                    for (int n = 0; n < NT; n++) mma_f16(acc[n][2 * w + u], f, pb[h][n][0], pb[h][n][1]);
                                }
                        }
                    }
                }
                __syncwarp();
                out.next();
                if (at * KEYS < cur.hi)
                    issue(cur, at++, in);
                else if (nat * KEYS < nxt.hi)
                    issue(nxt, nat++, in);
                else
                    flight--;
            }
            bool out_of_range = false;
            // the chunk's result: lane (g, i) holds dimensions 16 g .. + 15 of rows 2 i and 2 i + 1
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float x = l[n][c];
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    x += __shfl_xor_sync(0xffffffffu, x, 8);
                    x += __shfl_xor_sync(0xffffffffu, x, 16);
                    const int row = 8 * n + 2 * i + c;
                    if (row >= cur.n_rows) continue;
                    if (cur.chunks == 1) {
#pragma unroll
                        for (int j = 0; j < 8; j += 2)
                            out_of_range |= store_row<T>(a, cur.start, cur.kvh, cur.row0 + row, 4 * g + j / 2,
                                                         make_float4(acc[n][j][c], acc[n][j][c + 2], acc[n][j + 1][c], acc[n][j + 1][c + 2]), x);
                    } else {
                        const int64_t p = ((int64_t)cur.item * kvh_n + cur.kvh) * a.rows + row;
                        float4* dst = (float4*)(a.part_o + p * PG_DIM + 16 * g);
#pragma unroll
                        for (int j = 0; j < 8; j += 2)
                            dst[j / 2] = make_float4(acc[n][j][c], acc[n][j][c + 2], acc[n][j + 1][c], acc[n][j + 1][c + 2]);
                        if (g == 0) a.part_ml[p] = make_float2(m[n][c], x);
                    }
                }
            if (out_of_range) paged_report(a.b.status, JV_ERR_NUMERIC, PS_ATTN_VALUE);
        }
        // what the next item still lacks of its first stages (all of them after an item without keys)
        cur = nxt;
        at = nat;
        for (; flight < STAGES && at * KEYS < cur.hi; flight++) issue(cur, at++, in);
    }
}

// Joins the chunks of small requests: one CTA per (row, request, KV head), its warps over the chunks with a
// running reference each, four chunks' loads in flight. Latency-bound: a request of more than KJ_FEW chunks takes 16
// warps, the others 4. That goes by the request's own chunks, since the order of the sums, and with it the last
// bits, goes by the warps; the batch's bounds only say how many the CTAs have (with 4 for tables of up to 512 pages,
// which cannot hold more than KJ_FEW chunks, fewer warps are idle).
constexpr int KJ_FEW = 128;
// The row's chunks by WAYS warps.
template <class T, int WAYS>
__device__ __forceinline__ void join_chunks(const AttnKArgs& a, const RequestRows& rr, int row, int kvh, int chunks, int64_t p0,
                                            float4 (*so)[32], float2* sl) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t step = (int64_t)a.c.kv_heads * a.rows;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    for (int c0 = warp < WAYS ? warp : chunks; c0 < chunks; c0 += 4 * WAYS) {
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int c = c0 + k * WAYS;
            const bool in = c < chunks;
            ml[k] = in ? a.part_ml[p0 + c * step] : make_float2(-INFINITY, 0.f);
            x[k] = in ? *(const float4*)(a.part_o + (p0 + c * step) * PG_DIM + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float mn = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
        const float ref = mn == -INFINITY ? 0.f : mn, f0 = ex2(m - ref);
        m = mn;
        l *= f0;
        o.x *= f0, o.y *= f0, o.z *= f0, o.w *= f0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = ex2(ml[k].x - ref);
            l = fmaf(ml[k].y, f, l);
            o.x = fmaf(x[k].x, f, o.x), o.y = fmaf(x[k].y, f, o.y), o.z = fmaf(x[k].z, f, o.z), o.w = fmaf(x[k].w, f, o.w);
        }
    }
    if (warp < WAYS) {
        so[warp][lane] = o;
        if (lane == 0) sl[warp] = make_float2(m, l);
    }
    __syncthreads();
    if (warp) return;
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAYS; w++) m = fmaxf(m, sl[w].x);
    const float ref = m == -INFINITY ? 0.f : m;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < WAYS; w++) {
        const float f = ex2(sl[w].x - ref);
        const float4 x = so[w][lane];
        l = fmaf(sl[w].y, f, l);
        o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
    }
    if (store_row<T>(a, rr.start, kvh, row, lane, o, l)) paged_report(a.b.status, JV_ERR_NUMERIC, PS_ATTN_VALUE);
}
template <class T, int KJ_WARPS>
__global__ void __launch_bounds__(KJ_WARPS * 32) k_kv8_join(AttnKArgs a) {
    __shared__ float4 so[KJ_WARPS][32];
    __shared__ float2 sl[KJ_WARPS];
    pdl_wait();
    const int row = blockIdx.x, request = blockIdx.y, kvh = blockIdx.z;
    RequestRows rr;
    const int first = a.v.first[request];  // asked for together with the rows
    if (!request_rows(a.b, request, rr)) return;
    const int n_rows = rr.n_new * a.b.group, chunks = pg_chunks(rr.len, n_rows);
    if (n_rows > PG_SMALL_ROWS || row >= n_rows || chunks < 2) return;
    const int item0 = first + row / PG_ROW_TILE * chunks;
    if (first < 0 || item0 + chunks > a.v.small_cap) return;
    const int64_t p0 = ((int64_t)item0 * a.c.kv_heads + kvh) * a.rows + row % PG_ROW_TILE;
    if (KJ_WARPS > 4 && chunks > KJ_FEW)
        join_chunks<T, KJ_WARPS>(a, rr, row, kvh, chunks, p0, so, sl);
    else
        join_chunks<T, 4>(a, rr, row, kvh, chunks, p0, so, sl);
}

// Query rows of a small item, and row tiles of a small request, at most.
int tile_rows(const jv_paged_batch& b) { return (int)std::min<int64_t>(PG_ROW_TILE, (int64_t)b.max_new * b.group); }
int small_rows(const jv_paged_batch& b) { return (int)std::min<int64_t>(PG_SMALL_ROWS, (int64_t)b.max_new * b.group); }

struct Workspace {
    int64_t o, ml, large_o, large_ml, bytes;
};
Workspace workspace(const jv_paged_batch& b, int kv_heads) {
    const PlanView v = plan_view(b);
    const int64_t small = v.small_cap * kv_heads * tile_rows(b), large = v.split_cap * kv_heads * 2 * PG_TILE;
    Workspace w;
    w.o = 0;
    w.ml = small * PG_DIM * 4;
    w.large_o = (w.ml + small * 8 + 15) & ~(int64_t)15;
    w.large_ml = w.large_o + large * PG_DIM * 4;
    w.bytes = w.large_ml + large * 8;
    return w;
}

// The cache as a 4-dimensional tensor of bytes, [page][kv head][K rows, V rows][128]; a box is the K or
// the V of `keys` tokens of one head. The encoder is looked up once through the runtime, so the library needs no link to libcuda.
CUtensorMap page_map(const jv_kv8_cache& c, int keys) {
    using Encode = decltype(&cuTensorMapEncodeTiled);
    static const Encode encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        JV_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r));
        if (!p || r != cudaDriverEntryPointSuccess) throw Error(JV_ERR_DEVICE, "the driver has no cuTensorMapEncodeTiled");
        return (Encode)p;
    }();
    CUtensorMap m;
    const cuuint64_t dims[4] = {PG_DIM, 2 * PG_TOKENS, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {PG_DIM, 2 * PG_PLANE, (cuuint64_t)c.page_bytes};
    const cuuint32_t box[4] = {PG_DIM, (cuuint32_t)keys, 1, 1}, ones[4] = {1, 1, 1, 1};
    const CUresult r = encode(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, c.data, dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error(JV_ERR_DEVICE, "cuTensorMapEncodeTiled failed with " + std::to_string((int)r));
    return m;
}

// The kernel's dynamic shared memory limit, once per kernel and device.
template <auto kernel>
void allow_smem(int bytes) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    JV_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (done.load() & bit) return;
    JV_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done.fetch_or(bit);
}

template <class T, int NT>
void launch_small(const AttnKArgs& a, int ctas, cudaStream_t s) {
    const CUtensorMap map = page_map(a.c, Ks<NT>::keys);
    allow_smem<k_kv8_small<T, NT>>(Ks<NT>::smem);
    launch_pdl(k_kv8_small<T, NT>, dim3(ctas), dim3(KS_WARPS * 32), Ks<NT>::smem, s, a, map);
    note_launch();
}

template <class T>
void launch(const AttnKArgs& a, cudaStream_t s) {
    int sms = 148, dev = 0;
    JV_CUDA(cudaGetDevice(&dev));
    JV_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const int64_t small = a.v.small_cap * a.c.kv_heads;
    const int ctas = (int)std::min<int64_t>((small + KS_WARPS - 1) / KS_WARPS, (a.rows <= 8 ? Ks<1>::ctas : Ks<2>::ctas) * sms);
    if (a.rows <= 8)
        launch_small<T, 1>(a, ctas, s);
    else
        launch_small<T, 2>(a, ctas, s);
    if (a.b.max_keys > PG_CHUNK) {
        const dim3 grid(small_rows(a.b), a.b.requests, a.c.kv_heads);
        if (a.b.max_blocks > KJ_FEW * 256 / PG_TOKENS)  // chunks of 256 keys and more
            launch_pdl(k_kv8_join<T, 16>, grid, dim3(16 * 32), 0, s, a);
        else
            launch_pdl(k_kv8_join<T, 4>, grid, dim3(4 * 32), 0, s, a);
        note_launch();
    }
}

}  // namespace
}  // namespace jv

using namespace jv;

extern "C" {

int64_t jv_kv8_attention_bytes(const jv_paged_batch* batch, int32_t kv_heads) {
    int64_t n = -1;
    paged_api([&] {
        check_batch(batch, false);
        if (kv_heads < 1 || kv_heads > 1024) throw Error(JV_ERR_ARG, "1 to 1024 KV heads");
        n = workspace(*batch, kv_heads).bytes;
    });
    return n;
}

int jv_kv8_attention(const jv_kv8_cache* cache, const jv_paged_batch* batch, int32_t type, const jv_heads* q, float scale,
                     int32_t window, void* ws, int64_t workspace_bytes, void* stream) {
    return paged_api([&] {
        check_cache(cache);
        check_batch(batch, true);
        if (batch->pages != cache->pages) throw Error(JV_ERR_ARG, "the batch and the cache have different numbers of pages");
        if (type != T_F16 && type != T_BF16) throw Error(JV_ERR_UNSUPPORTED, "attention takes F16 (1) or BF16 (30) queries");
        if (!q || !q->in || !q->out) throw Error(JV_ERR_ARG, "NULL buffer");
        if (q->heads != cache->kv_heads * batch->group)
            throw Error(JV_ERR_ARG, "q must have kv_heads * group heads");
        auto ok = [](const void* p, int64_t x, int64_t y) { return (uintptr_t)p % 16 == 0 && x % 8 == 0 && y % 8 == 0 && x >= 0 && y >= 0; };
        if (!ok(q->in, q->in_token, q->in_head) || !ok(q->out, q->out_token, q->out_head))
            throw Error(JV_ERR_ARG, "attention: q and its output need 16-byte aligned rows (strides that are multiples of 8)");
        check_rows(q, "attention", PG_DIM, 1);  // within a token: max_tokens is only a bound
        if (q->in == q->out && (q->in_token != q->out_token || q->in_head != q->out_head))
            throw Error(JV_ERR_ARG, "attention: q in place must have the same strides in and out");
        if (window < 0) throw Error(JV_ERR_ARG, "attention: window is negative");
        if (!std::isfinite(scale)) throw Error(JV_ERR_ARG, "attention: scale must be finite");
        const Workspace w = workspace(*batch, cache->kv_heads);
        if (workspace_bytes < w.bytes) throw Error(JV_ERR_ARG, "attention: the workspace is smaller than jv_kv8_attention_bytes");
        if (!ws || (uintptr_t)ws % 16) throw Error(JV_ERR_ARG, "attention: the workspace must be 16-byte aligned");
        if (plan_view(*batch).large_cap > INT32_MAX / cache->kv_heads)
            throw Error(JV_ERR_RANGE, "attention: too many tokens and KV heads for one call");
        OnDeviceOf dev(cache->data);
        AttnKArgs a{};
        a.c = *cache;
        a.b = *batch;
        a.v = plan_view(*batch);
        a.q = *q;
        a.scale = scale * KA_LOG2E;
        a.window = window;
        a.part_o = (float*)((char*)ws + w.o);
        a.part_ml = (float2*)((char*)ws + w.ml);
        a.rows = tile_rows(*batch);
        a.large_o = (float*)((char*)ws + w.large_o);
        a.large_ml = (float2*)((char*)ws + w.large_ml);
        if (type == T_F16)
            launch<__half>(a, (cudaStream_t)stream);
        else
            launch<__nv_bfloat16>(a, (cudaStream_t)stream);
        if (a.v.large_cap > 0) launch_kv8_large(a, type, (cudaStream_t)stream);
    });
}

}  // extern "C"
