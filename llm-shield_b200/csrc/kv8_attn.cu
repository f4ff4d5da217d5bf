// kv8_attn.cu — grouped-query attention over the 8-bit paged cache (jv_kv8_attention).
//
// o = sum_j softmax_j(scale q . k_j) v_j with k_j = ks(j) kint_j and v_j = vs(j) vint_j, where ks and vs
// are the scales of key j's block of 16. The scales never touch the matrices: with
//   e_j = scale ks(j) (q . kint_j) + log2 vs(j)   (in log2 units),   w_j = 2^(e_j - M),   M >= max e_j - 8
// the output is  sum_j w_j vint_j / sum_j (w_j / vs(j)),  so the products run on exact integers (an
// int8 is exact in fp16), w_j <= 2^8 is the only rounded operand (fp16, half a step 2^-12), and sums, M
// and the softmax denominator are fp32. bf16 queries are taken to fp16 by a power of two per row.
//
// The products are mma.sync m16n8k16 with the keys on the 16-row side and the query rows (new token x
// head of the group) on the 8-column side: S^T = K Q^T, O^T = V^T P^T. The order of the 128
// dimensions inside a product is free, so a lane loads 16 consecutive int8 of its rows straight from
// the cache into fragments; S^T becomes the operand P^T by one movmatrix per 8 x 8 block.
#include <cmath>
#include <string>

#include <cuda_bf16.h>

#include "paged.h"

namespace jv {
namespace {

constexpr int KA_WARPS = 4;
constexpr int KA_THREADS = KA_WARPS * 32;
constexpr float KA_LOG2E = 1.4426950408889634f;

struct AttnKArgs {
    jv_kv8_cache c;
    jv_paged_batch b;
    PlanView v;
    jv_heads q;
    float scale;  // times log2 e
    int window;
    float* part_o;   // [small item][kv head][rows][128]
    float2* part_ml; // [small item][kv head][rows]
    int rows;        // query rows of a small item's partials
};

__device__ __forceinline__ float ex2f(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
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

template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t x);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t x) { return __half22float2(*(const __half2*)&x); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t x) {
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

// Rows [row0, row0 + 8 NT) of a request's query rows (row = new token * group + head of the group)
// against keys [k_lo, k_hi) of one KV head, by one CTA. The warps take the 16-key tiles in turn and
// are joined in shared memory. Leaves acc / m / l joined in shared memory: O[row][dim], ml[row].
template <class T, int NT>
struct Smem {
    float o[KA_WARPS][8 * NT][PG_DIM + 4];
    float m[KA_WARPS][8 * NT], l[KA_WARPS][8 * NT];
};

template <class T, int NT>
__device__ __forceinline__ void attend(const AttnKArgs& a, Smem<T, NT>& sm, const RequestRows& rr, int request, int kvh,
                                       int row0, int k_lo, int k_hi) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, i = lane & 3;
    const int group = a.b.group, n_rows = rr.n_new * group;
    // B fragments of Q^T: lane (g, i) holds row g's dimensions 16 i .. + 15 and 64 + 16 i .. + 15
    uint32_t qf[NT][16];
    float qs[NT][2];         // per accumulator column 2 i, 2 i + 1: the scale of its row
    int lo_key[NT][2], hi_key[NT][2];  // visible keys of that row
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int row = row0 + 8 * n + g;
        float f = 1.f;
        if (row < n_rows) {
            const T* src = (const T*)a.q.in + (int64_t)(rr.start + row / group) * a.q.in_token +
                           (int64_t)(kvh * group + row % group) * a.q.in_head + 16 * i;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint4 x = *(const uint4*)(src + 64 * j + 8 * e);
                    qf[n][8 * j + 4 * e] = x.x, qf[n][8 * j + 4 * e + 1] = x.y;
                    qf[n][8 * j + 4 * e + 2] = x.z, qf[n][8 * j + 4 * e + 3] = x.w;
                }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e++) qf[n][e] = 0;
        }
        if (std::is_same<T, __nv_bfloat16>::value) {
            // bf16 -> fp16 times a power of two that puts the row's largest magnitude in [2^13, 2^14): exact
            // but for values 2^27 below it
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float2 x = unpack2<T>(qf[n][e]);
                amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = min(max((int)((__float_as_uint(amax) >> 23) & 0xff), 14), 254);  // 2^(ex - 127) <= amax
            const float up = __uint_as_float((uint32_t)(267 - ex) << 23);  // 2^(13 - (ex - 127))
            f = 1.f / up;
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float2 x = unpack2<T>(qf[n][e]);
                qf[n][e] = pack2<__half>(x.x * up, x.y * up);
            }
        }
        f *= a.scale;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int col = 2 * i + e, r = row0 + 8 * n + col;
            qs[n][e] = __shfl_sync(0xffffffffu, f, 4 * col);
            const int pos = rr.len - rr.n_new + r / group;
            hi_key[n][e] = r < n_rows ? pos + 1 : 0;
            lo_key[n][e] = a.window > 0 ? max(0, pos + 1 - a.window) : 0;
        }
    }
    float acc[NT][8][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[n][j][e] = 0.f;
    }
    const int32_t* table = a.b.block_table + (int64_t)request * a.b.max_blocks;
    for (int t = k_lo / PG_BLOCK + warp; t * PG_BLOCK < k_hi; t += KA_WARPS) {
        const int key0 = t * PG_BLOCK;
        const int page = table[key0 / PG_TOKENS];
        if ((unsigned)page >= (unsigned)a.c.pages) {
            if (lane == 0) paged_report(a.b.status, JV_ERR_RANGE, PS_ATTN_PAGE);
            continue;
        }
        const char* kp = (const char*)a.c.data + (int64_t)page * a.c.page_bytes + (int64_t)kvh * 2 * PG_PLANE +
                         (key0 % PG_TOKENS) * PG_DIM;
        const char* vp = kp + PG_PLANE;
        const float* sp = a.c.scales + (int64_t)page * a.c.scale_stride + kvh * 8 + (key0 % PG_TOKENS) / PG_BLOCK;
        const float ks = sp[0];
        float vs = sp[4];
        uint4 kr[2][2], vr[4];
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int j = 0; j < 2; j++) kr[r][j] = *(const uint4*)(kp + (g + 8 * r) * PG_DIM + 64 * j + 16 * i);
#pragma unroll
        for (int r = 0; r < 4; r++) vr[r] = *(const uint4*)(vp + (2 * i + (r & 1) + 8 * (r >> 1)) * PG_DIM + 16 * g);
        if (!(vs > 0.f)) vs = 1.f;  // a block of zeros
        const float lvs = log2f(vs), ivs = 1.f / vs;
        // S^T
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t w0[4] = {kr[0][j].x, kr[0][j].y, kr[0][j].z, kr[0][j].w};
            const uint32_t w1[4] = {kr[1][j].x, kr[1][j].y, kr[1][j].z, kr[1][j].w};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t x0 = w0[w] ^ 0x80808080u, x1 = w1[w] ^ 0x80808080u;
                const uint32_t f[4] = {pair_f16(x0, 0x4140), pair_f16(x1, 0x4140), pair_f16(x0, 0x4342), pair_f16(x1, 0x4342)};
#pragma unroll
                for (int n = 0; n < NT; n++) mma_f16(s[n], f, qf[n][8 * j + 2 * w], qf[n][8 * j + 2 * w + 1]);
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            float e[4], mx[2];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int key = key0 + g + 8 * (x >> 1), c = x & 1;
                e[x] = fmaf(s[n][x], ks * qs[n][c], lvs);
                if (key >= hi_key[n][c] || key < lo_key[n][c]) e[x] = -INFINITY;
            }
            float alpha[2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                mx[c] = fmaxf(e[c], e[c + 2]);
                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 4));
                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 8));
                mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], 16));
                const float mn = fmaxf(m[n][c], mx[c]);
                const float ref = mn == -INFINITY ? 0.f : mn;
                alpha[c] = ex2f(m[n][c] - ref);
                m[n][c] = mn;
                e[c] = ex2f(e[c] - ref);
                e[c + 2] = ex2f(e[c + 2] - ref);
                l[n][c] = fmaf(l[n][c], alpha[c], (e[c] + e[c + 2]) * ivs);
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int x = 0; x < 4; x++) acc[n][j][x] *= alpha[x & 1];
            }
            pb[n][0] = movmatrix_trans(pack2<__half>(e[0], e[1]));
            pb[n][1] = movmatrix_trans(pack2<__half>(e[2], e[3]));
        }
        // O^T += V^T P^T: dimension 16 g + 2 j is the tile's row g, 16 g + 2 j + 1 its row g + 8
        const uint32_t va[4] = {vr[0].x, vr[0].y, vr[0].z, vr[0].w}, vb[4] = {vr[1].x, vr[1].y, vr[1].z, vr[1].w};
        const uint32_t vc[4] = {vr[2].x, vr[2].y, vr[2].z, vr[2].w}, vd[4] = {vr[3].x, vr[3].y, vr[3].z, vr[3].w};
#pragma unroll
        for (int w = 0; w < 4; w++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const uint32_t sel = u ? 0x7362 : 0x5140;
                const uint32_t lo = __byte_perm(va[w], vb[w], sel) ^ 0x80808080u, hi = __byte_perm(vc[w], vd[w], sel) ^ 0x80808080u;
                const uint32_t f[4] = {pair_f16(lo, 0x4140), pair_f16(lo, 0x4342), pair_f16(hi, 0x4140), pair_f16(hi, 0x4342)};
#pragma unroll
                for (int n = 0; n < NT; n++) mma_f16(acc[n][2 * w + u], f, pb[n][0], pb[n][1]);
            }
    }
    // join the warps
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
            l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
            const int row = 8 * n + 2 * i + c;
            if (g == 0) {
                sm.m[warp][row] = m[n][c];
                sm.l[warp][row] = l[n][c];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float2* dst = (float2*)&sm.o[warp][row][16 * g + 2 * j];
                *dst = make_float2(acc[n][j][c], acc[n][j][c + 2]);
            }
        }
    __syncthreads();
}

// Row r of the joined warps, dimensions 4 d4 .. + 3: unnormalised values, reference and denominator.
template <class T, int NT>
__device__ __forceinline__ float4 joined(const Smem<T, NT>& sm, int r, int d4, float& m, float& l) {
    m = -INFINITY;
#pragma unroll
    for (int w = 0; w < KA_WARPS; w++) m = fmaxf(m, sm.m[w][r]);
    const float ref = m == -INFINITY ? 0.f : m;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    l = 0.f;
#pragma unroll
    for (int w = 0; w < KA_WARPS; w++) {
        const float f = ex2f(sm.m[w][r] - ref);
        const float4 x = *(const float4*)&sm.o[w][r][4 * d4];
        l = fmaf(sm.l[w][r], f, l);
        o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
    }
    return o;
}

template <class T>
__device__ __forceinline__ void store_row(const AttnKArgs& a, const RequestRows& rr, int kvh, int row, int d4, float4 o, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // no visible key: zeros (a NaN stays one)
    T* dst = (T*)a.q.out + (int64_t)(rr.start + row / a.b.group) * a.q.out_token +
             (int64_t)(kvh * a.b.group + row % a.b.group) * a.q.out_head + 4 * d4;
    *(uint2*)dst = make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
}

// Small requests: persistent CTAs over (chunk of a request, KV head).
template <class T, int NT>
__global__ void __launch_bounds__(KA_THREADS) k_kv8_small(AttnKArgs a) {
    __shared__ __align__(16) Smem<T, NT> sm;
    const int kvh_n = a.c.kv_heads;
    const int64_t n = (int64_t)min((int64_t)max(a.v.head[0], 0), a.v.small_cap) * kvh_n;
    for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
        const int item = (int)(w / kvh_n), kvh = (int)(w % kvh_n);
        const int4 it = a.v.small_items[item];
        RequestRows rr;
        if (!request_rows(a.b, it.x, rr)) continue;
        const int n_rows = rr.n_new * a.b.group;
        if (n_rows > 8 * NT || n_rows > a.rows) continue;
        const int ck = pg_chunk_keys(max(rr.len, 1));
        int lo = it.y * ck, hi = min(rr.len, lo + ck);
        if (a.window > 0) lo = max(lo, max(0, rr.len - rr.n_new + 1 - a.window));
        attend<T, NT>(a, sm, rr, it.x, kvh, 0, lo, hi);
        for (int e = threadIdx.x; e < n_rows * 32; e += KA_THREADS) {
            const int r = e >> 5, d4 = e & 31;
            float m, l;
            const float4 o = joined<T, NT>(sm, r, d4, m, l);
            if (it.z == 1) {
                store_row<T>(a, rr, kvh, r, d4, o, l);
            } else {
                const int64_t p = ((int64_t)item * kvh_n + kvh) * a.rows + r;
                *(float4*)(a.part_o + p * PG_DIM + 4 * d4) = o;
                if (d4 == 0) a.part_ml[p] = make_float2(m, l);
            }
        }
        __syncthreads();
    }
}

// Joins the chunks of small requests: one CTA per (request, KV head, row), its warps over the chunks.
template <class T>
__global__ void __launch_bounds__(256) k_kv8_join(AttnKArgs a) {
    __shared__ float4 so[8][32];
    __shared__ float sl[8];
    const int request = blockIdx.x, kvh = blockIdx.y, row = blockIdx.z;
    RequestRows rr;
    if (!request_rows(a.b, request, rr)) return;
    const int n_rows = rr.n_new * a.b.group, chunks = pg_chunks(rr.len);
    if (n_rows > PG_SMALL_ROWS || row >= n_rows || chunks < 2) return;
    const int first = a.v.first[request];
    if (first < 0 || first + chunks > a.v.small_cap) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t p0 = ((int64_t)first * a.c.kv_heads + kvh) * a.rows + row, step = (int64_t)a.c.kv_heads * a.rows;
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 32) m = fmaxf(m, a.part_ml[p0 + c * step].x);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float ref = m == -INFINITY ? 0.f : m;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 4
    for (int c = warp; c < chunks; c += 8) {
        const float2 ml = a.part_ml[p0 + c * step];
        const float4 x = *(const float4*)(a.part_o + (p0 + c * step) * PG_DIM + 4 * lane);
        const float f = ex2f(ml.x - ref);
        l = fmaf(ml.y, f, l);
        o.x = fmaf(x.x, f, o.x), o.y = fmaf(x.y, f, o.y), o.z = fmaf(x.z, f, o.z), o.w = fmaf(x.w, f, o.w);
    }
    so[warp][lane] = o;
    if (lane == 0) sl[warp] = l;
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < 8; w++) {
        const float4 x = so[w][lane];
        o.x += x.x, o.y += x.y, o.z += x.z, o.w += x.w;
        l += sl[w];
    }
    store_row<T>(a, rr, kvh, row, lane, o, l);
}

// Large requests: one CTA per (tile of 16 query rows, KV head), over all its keys.
template <class T>
__global__ void __launch_bounds__(KA_THREADS) k_kv8_large(AttnKArgs a) {
    __shared__ __align__(16) Smem<T, 2> sm;
    const int kvh_n = a.c.kv_heads;
    const int64_t n = (int64_t)min((int64_t)max(a.v.head[1], 0), a.v.large_cap) * kvh_n;
    for (int64_t w = blockIdx.x; w < n; w += gridDim.x) {
        const int kvh = (int)(w % kvh_n);
        const int4 it = a.v.large_items[w / kvh_n];
        RequestRows rr;
        if (!request_rows(a.b, it.x, rr)) continue;
        const int n_rows = rr.n_new * a.b.group, row0 = it.y * PG_TILE_ROWS;
        if (row0 < 0 || row0 >= n_rows) continue;
        const int rows = min(PG_TILE_ROWS, n_rows - row0);
        const int first = rr.len - rr.n_new + row0 / a.b.group, last = rr.len - rr.n_new + (row0 + rows - 1) / a.b.group;
        attend<T, 2>(a, sm, rr, it.x, kvh, row0, a.window > 0 ? max(0, first + 1 - a.window) : 0, max(0, last + 1));
        for (int e = threadIdx.x; e < rows * 32; e += KA_THREADS) {
            float m, l;
            const float4 o = joined<T, 2>(sm, e >> 5, e & 31, m, l);
            store_row<T>(a, rr, kvh, row0 + (e >> 5), e & 31, o, l);
        }
        __syncthreads();
    }
}

int small_rows(const jv_paged_batch& b) { return (int)std::min<int64_t>(PG_SMALL_ROWS, (int64_t)b.max_new * b.group); }

struct Workspace {
    int64_t o, ml, bytes;
};
Workspace workspace(const jv_paged_batch& b, int kv_heads) {
    const int64_t n = (b.requests + b.max_keys / 256) * kv_heads * small_rows(b);
    return {0, n * PG_DIM * 4, n * (PG_DIM * 4 + 8)};
}

template <class T>
void launch(const AttnKArgs& a, cudaStream_t s) {
    int sms = 148, dev = 0;
    JV_CUDA(cudaGetDevice(&dev));
    JV_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const int64_t small = a.v.small_cap * a.c.kv_heads, large = a.v.large_cap * a.c.kv_heads;
    if (a.rows <= 8)
        k_kv8_small<T, 1><<<(unsigned)std::min<int64_t>(small, 4 * sms), KA_THREADS, 0, s>>>(a);
    else
        k_kv8_small<T, 2><<<(unsigned)std::min<int64_t>(small, 4 * sms), KA_THREADS, 0, s>>>(a);
    JV_CUDA(cudaGetLastError());
    note_launch();
    if (a.b.max_keys > 256) {
        k_kv8_join<T><<<dim3(a.b.requests, a.c.kv_heads, a.rows), 256, 0, s>>>(a);
        JV_CUDA(cudaGetLastError());
        note_launch();
    }
    if ((int64_t)a.b.max_new * a.b.group > PG_SMALL_ROWS) {
        k_kv8_large<T><<<(unsigned)std::min<int64_t>(large, 4 * sms), KA_THREADS, 0, s>>>(a);
        JV_CUDA(cudaGetLastError());
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
        a.rows = small_rows(*batch);
        if (type == T_F16)
            launch<__half>(a, (cudaStream_t)stream);
        else
            launch<__nv_bfloat16>(a, (cudaStream_t)stream);
    });
}

}  // extern "C"
