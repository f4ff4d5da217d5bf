// kv8_attn_tc.cu — attention over the 8-bit paged cache for requests of many query rows (prompts and
// their chunks), on the 5th-generation tensor cores. The mathematics is kv8_attn.cu's: integer keys and
// values, their scales in the exponent and in the denominator.
//
// One CTA = one KV head x a pair of query tiles A and B of 128 rows (128 / group tokens x the group's heads),
// which share every block of 128 keys; per tile and block
//   S = Q K^T   tcgen05.mma kind::f16, M = N = K = 128, S in TMEM (fp32)
//   w = 2^(e - M) as fp16 to shared memory (a row per thread, M moves only past 2^8)
//   O += W V    (V MN-major)
// TMEM: O_A, O_B, S_A, S_B, 128 columns each. A softmax hands its S columns back as soon as it has them in
// registers, so the next block's S runs under its exponentials, and each tile has its own W. (W over S in TMEM
// would save a third of the shared-memory traffic. It was measured before the packed arithmetic, the register split
// and the halves below: 230 us, 213 with the tiles taking turns, where W in shared memory took 219 at that
// point; not since.) A prompt of 4095 tokens, 32 / 8 heads: 183 us, 750 TFLOP/s of visible work, about 4,700 cycles a
// block of the two tiles, of which a softmax waits 950 for products. The exponential unit is busy for 2,048 of
// them, the tensor pipe for 2,048 and shared memory, with 384 KB of operands, weights and converted keys and
// values, for 3,072; with less work in the softmax a block took no fewer, so what is left is the products' way
// through shared memory and the hand-overs around them.
// Warps 0-3 and 4-7: the softmax and output of tiles A and B. Warps 8-11: convert the cache's int8 to fp16
// operands (K as b + 128 in subnormals, one byte permute; V signed), two stages of K and one of V, in the
// order K(b + 1), V(b), with the next blocks' bytes already in registers. Warps 12 and 13: issue tile A's and
// B's products. Registers are moved from the issuers to the softmax (128 at launch: 168 + 168 + 128 + 48 = 4 x
// 128). Every wait is bounded; on expiry the role records its site and stops.
#include <atomic>

#include <cuda_bf16.h>

#include "paged.h"
#include "tc_common.cuh"

namespace jv {
namespace {

constexpr int KT_THREADS = 512;
constexpr int KT_KEYS = 128;
constexpr int KT_TILE = 128 * 128 * 2;  // one fp16 operand tile
constexpr int KT_SLOTS = 4;             // blocks whose scales are kept
constexpr int KT_SMEM = 7 * KT_TILE + KT_SLOTS * 128 + 256 + 1024;

enum KtRole : int { KR_CONVERT_K = 0, KR_CONVERT_V = 1, KR_ISSUE = 2, KR_SOFTMAX = 3 };

template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

struct KtItem {
    RequestRows rr;
    int tt;               // tokens per tile
    int t0[2], nt[2];     // first token (of the request's new ones) and tokens of each tile
    int b0[2], b1[2];     // its blocks
    int lo, hi;           // blocks of the CTA
};

// 16 int8 of one row (dimensions 16 j ..) as 32 bytes of fp16 into a [128][128] operand tile. Eight lanes that
// store together hold four j of two neighbouring rows: eight different chunks.
template <bool SIGNED>
__device__ __forceinline__ void convert16(uint32_t tile, int row, int j, uint4 raw) {
    const uint32_t w[4] = {raw.x ^ 0x80808080u, raw.y ^ 0x80808080u, raw.z ^ 0x80808080u, raw.w ^ 0x80808080u};
    uint32_t h[8];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t fill = SIGNED ? 0x64646464u : 0u;
        h[2 * e] = __byte_perm(w[e], fill, 0x4140);
        h[2 * e + 1] = __byte_perm(w[e], fill, 0x4342);
        if (SIGNED) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const __half2 x = __hsub2(*(const __half2*)&h[2 * e + k], __floats2half2_rn(1152.f, 1152.f));
                h[2 * e + k] = *(const uint32_t*)&x;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; k++)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};\n" ::"r"(tile + tile_off(row, 2 * j + k)), "r"(h[4 * k]), "r"(h[4 * k + 1]),
                     "r"(h[4 * k + 2]), "r"(h[4 * k + 3])
                     : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// Packed fp32 pairs (a register pair each).
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float2 unpack_f32x2(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}

template <class T>
__global__ void __launch_bounds__(KT_THREADS, 1) k_kv8_large(AttnKArgs a) {
    extern __shared__ uint8_t kt_raw[];
    uint8_t* sm = kt_raw + ((1024u - (s_addr(kt_raw) & 1023u)) & 1023u);
    // Q_A, Q_B, two K, V, W_A, W_B
    const uint32_t Qs = s_addr(sm), Ks = Qs + 2 * KT_TILE, Vs = Qs + 4 * KT_TILE;
    float4* scales = (float4*)(sm + 7 * KT_TILE);  // [slot][8]: ks, log2 vs, 1 / vs of 16 keys
    uint64_t* bars = (uint64_t*)(sm + 7 * KT_TILE + KT_SLOTS * 128);
    const uint32_t k_full = s_addr(bars), k_empty = k_full + 16, q_full = k_full + 32, s_full = k_full + 48;
    const uint32_t s_free = k_full + 64, p_full = k_full + 80, o_done = k_full + 96, v_full = k_full + 112, v_empty = k_full + 120;
    uint32_t* tslot = (uint32_t*)(bars + 16);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    pdl_wait();
    pdl_launch_dependents();
    const int kvh_n = a.c.kv_heads, kvh = blockIdx.x % kvh_n, index = blockIdx.x / kvh_n;
    // in the lists' bounds, as the grid is; all at once, since every load that waits for another costs 700 cycles
    const int4 item = a.v.large_items[index], rows = a.v.large_rows[index];
    if (index >= a.v.head[1]) return;
    const int group = a.b.group, splits = item.w & 255, place = item.w >> 8;
    KtItem it;
    it.rr.start = rows.x, it.rr.n_new = rows.y, it.rr.len = rows.z;
    if (item.x < 0 || item.x >= a.b.requests || !rows_in_bounds(a.b, rows.x, rows.y, rows.z)) return;
    it.tt = PG_TILE / group;
    const int total_blocks = (int)(((int64_t)it.rr.len + KT_KEYS - 1) / KT_KEYS);
    const int per = splits > 0 ? (total_blocks + splits - 1) / splits : 0;
    if (item.y < 0 || item.z < 0 || item.z >= splits || (splits > 1 && (place < 0 || place >= a.v.split_cap)) || (int64_t)item.y * 2 * it.tt >= it.rr.n_new) return;
    const int s0 = min(item.z * per, total_blocks), s1 = min(s0 + per, total_blocks);
    it.lo = 1 << 30, it.hi = 0;
#pragma unroll
    for (int x = 0; x < 2; x++) {
        it.t0[x] = item.y * 2 * it.tt + x * it.tt;
        it.nt[x] = max(0, min(it.tt, it.rr.n_new - it.t0[x]));
        const int first = it.rr.len - it.rr.n_new + it.t0[x], last = first + it.nt[x] - 1;
        it.b1[x] = it.nt[x] > 0 && last >= 0 ? min(s1, last / KT_KEYS + 1) : 0;
        it.b0[x] = max(s0, a.window > 0 ? max(0, first + 1 - a.window) / KT_KEYS : 0);
        if (it.b0[x] >= it.b1[x]) it.b0[x] = it.b1[x] = 0;
        if (it.b0[x] < it.b1[x]) it.lo = min(it.lo, it.b0[x]), it.hi = max(it.hi, it.b1[x]);
    }
    if (it.lo > it.hi) it.lo = it.hi;

    // The first loads from the pages' table, on their way while the CTA sets up.
    const int32_t* table = a.b.block_table + (int64_t)item.x * a.b.max_blocks;
    const int pages = (int)(((int64_t)it.rr.len + PG_TOKENS - 1) / PG_TOKENS);
    // the two pages of a block; -1 where the request has none
    auto page_of = [&](int b, int h) {
        const int p = 2 * b + h;
        if (b >= it.hi || p >= pages) return -1;
        const int id = table[p];
        if ((unsigned)id >= (unsigned)a.c.pages) {
            if (lane == 0) paged_report(a.b.status, JV_ERR_RANGE, PS_ATTN_PAGE);
            return -1;
        }
        return id;
    };
    int p0 = -1, p1 = -1, n0 = -1, n1 = -1;  // pages of the block whose K is next, and of the one after it
    if (warp >= 8 && warp < 12) p0 = page_of(it.lo, 0), p1 = page_of(it.lo, 1), n0 = page_of(it.lo + 1, 0), n1 = page_of(it.lo + 1, 1);
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(k_full + 8 * i, 4);
            mbar_init(k_empty + 8 * i, 2);
            mbar_init(s_free + 8 * i, 4);
            mbar_init(q_full + 8 * i, 4);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 4);
            mbar_init(o_done + 8 * i, 1);
        }
        mbar_init(v_full, 4);
        mbar_init(v_empty, 2);
        fence_barrier_init();
    }
    if (warp == 12) tmem_alloc(s_addr(tslot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    int* err = a.b.status;

    if (warp >= 12) {
        reg_dec<48>();
        if (warp < 14) {
            // ------------------------------------------------ issue the products of one tile
            const int x = warp - 12;
            const uint32_t id_s = idesc_f16(KT_KEYS, PG_TILE), id_o = idesc_f16(PG_DIM, PG_TILE) | (1u << 16);
            const uint32_t q = Qs + x * KT_TILE, w = Qs + (5 + x) * KT_TILE, o = tmem + (uint32_t)(x * 128),
                           d = tmem + 256u + (uint32_t)(x * 128);
            const int b0 = it.b0[x], b1 = it.b1[x];
            auto all_wait = [&](uint32_t bar, uint32_t parity) { return warp_wait(bar, parity); };
            // The other tile's block n: released at once, but not before it is there (a release counts for the
            // stage's current use).
            auto skip = [&](int n) {
                if (!all_wait(k_full + 8 * (n & 1), (uint32_t)((n >> 1) & 1)) || !all_wait(v_full, (uint32_t)(n & 1))) return false;
                if (lane == 0) {
                    mbar_arrive(k_empty + 8 * (n & 1));
                    mbar_arrive(v_empty);
                }
                __syncwarp();
                return true;
            };
            auto issue_s = [&](int b) {
                const int n = b - it.lo;
                if (!all_wait(k_full + 8 * (n & 1), (uint32_t)((n >> 1) & 1))) return false;
                if (b > b0 && !all_wait(s_free + 8 * x, (uint32_t)((b - 1 - b0) & 1))) return false;
                tc_fence_after();
                const uint32_t k = Ks + (n & 1) * KT_TILE;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < 8; kk++) {
                        const uint32_t off = (uint32_t)((kk >> 2) * 16384 + (kk & 3) * 32);
                        umma(d, sdesc(q + off), sdesc(k + off), id_s, kk > 0 ? 1u : 0u);
                    }
                    umma_commit(s_full + 8 * x);
                    umma_commit(k_empty + 8 * (n & 1));
                }
                __syncwarp();
                return true;
            };
            auto issue_o = [&](int b) {
                const int n = b - it.lo;
                if (!all_wait(p_full + 8 * x, (uint32_t)((b - b0) & 1)) || !all_wait(v_full, (uint32_t)(n & 1))) return false;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < 8; kk++) {
                        const uint32_t off = (uint32_t)((kk >> 2) * 16384 + (kk & 3) * 32);
                        umma(o, sdesc(w + off), sdesc_mn(Vs + kk * 2048), id_o, b > b0 || kk > 0 ? 1u : 0u);
                    }
                    umma_commit(o_done + 8 * x);
                    umma_commit(v_empty);
                }
                __syncwarp();
                return true;
            };
            bool ok = true;
            int n = 0;
            if (b0 < b1) {
                for (; n < b0 - it.lo && ok; n++) ok = skip(n);
                ok = ok && warp_wait(q_full + 8 * x, 0) && issue_s(b0);
                for (int b = b0; b < b1 && ok; b++, n++) {
                    if (b + 1 < b1) ok = issue_s(b + 1);
                    ok = ok && issue_o(b);
                }
            }
            for (; n < it.hi - it.lo && ok; n++) ok = skip(n);
            if (!ok && lane == 0) paged_report(err, JV_ERR_DEVICE_TIMEOUT, PS_ATTN_TC + KR_ISSUE);
        }
    } else if (warp >= 8) {
        reg_dec<128>();
        // ---------------------------------------------------- int8 -> fp16 operands
        const int t = tid - 256, j0 = t & 3, r0 = t >> 2;  // 16 bytes j0 and j0 + 4 of rows r0 + 32 k
        uint4 kr[8], vr[8];
        auto load = [&](uint4 (&r)[8], int p0, int p1, int plane) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int id = k < 4 ? p0 : p1;  // piece k: row r0 + 32 (k / 2), bytes 16 (j0 + 4 (k & 1))
                r[k] = make_uint4(0, 0, 0, 0);
                if (id >= 0)
                    r[k] = *(const uint4*)((const char*)a.c.data + (int64_t)id * a.c.page_bytes + (int64_t)(2 * kvh + plane) * PG_PLANE +
                                           (r0 + 32 * ((k >> 1) & 1)) * PG_DIM + 16 * (j0 + 4 * (k & 1)));
            }
        };
        // Block n's keys and scales; its bytes are in kr, its pages p0 and p1. Loads the next block's.
        auto keys = [&](int n) {
            const int b = it.lo + n;
            float4 sc = make_float4(0.f, -INFINITY, 1.f, 0.f);  // keys without a page have no weight
            if (t < 8) {
                const int id = t < 4 ? p0 : p1;
                const int64_t key = (int64_t)b * KT_KEYS + t * PG_BLOCK;
                if (id >= 0 && key < it.rr.len) {
                    const float* s = a.c.scales + (int64_t)id * a.c.scale_stride + kvh * 8 + (t & 3);
                    const float vs = s[4] > 0.f ? s[4] : PG_ZERO_SCALE;
                    sc = make_float4(s[0], lg2_approx(vs), __frcp_rn(vs), 0.f);
                }
            }
            if (!warp_wait(k_empty + 8 * (n & 1), (uint32_t)((n >> 1) & 1) ^ 1u)) {
                if (lane == 0) paged_report(err, JV_ERR_DEVICE_TIMEOUT, PS_ATTN_TC + KR_CONVERT_K);
                return false;
            }
            if (t < 8) scales[(n & (KT_SLOTS - 1)) * 8 + t] = sc;
#pragma unroll
            for (int k = 0; k < 8; k++) convert16<false>(Ks + (n & 1) * KT_TILE, r0 + 32 * (k >> 1), j0 + 4 * (k & 1), kr[k]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full + 8 * (n & 1));
            p0 = n0, p1 = n1;
            load(kr, p0, p1, 0);
            n0 = page_of(b + 2, 0), n1 = page_of(b + 2, 1);
            return true;
        };
        load(kr, p0, p1, 0);
        load(vr, p0, p1, 1);
        const int blocks = it.hi - it.lo;
        bool ok = blocks == 0 || keys(0);
        for (int n = 0; n < blocks && ok; n++) {
            const int v0 = p0, v1 = p1;  // the pages of block n + 1
            if (n + 1 < blocks) ok = keys(n + 1);
            if (!ok) break;
            ok = warp_wait(v_empty, (uint32_t)(n & 1) ^ 1u);
            if (!ok) {
                if (lane == 0) paged_report(err, JV_ERR_DEVICE_TIMEOUT, PS_ATTN_TC + KR_CONVERT_V);
                break;
            }
#pragma unroll
            for (int k = 0; k < 8; k++) convert16<true>(Vs, r0 + 32 * (k >> 1), j0 + 4 * (k & 1), vr[k]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full);
            if (n + 1 < blocks) load(vr, v0, v1, 1);
        }
    } else {
        reg_inc<168>();
        // ---------------------------------------------------- softmax and output, a query row per thread
        const int x = warp >> 2, r = tid & 127;
        const int b0 = it.b0[x], b1 = it.b1[x], nt = it.nt[x], t0 = it.t0[x];
        const uint32_t per_row = (65536u + group - 1) / group;  // row / group for rows below 128
        auto token_of = [&](int row) { return (int)(((uint32_t)row * per_row) >> 16); };
        const int tok = token_of(r);
        const bool live = tok < nt;
        const int pos = it.rr.len - it.rr.n_new + t0 + tok;
        // rows of no token see everything: they are not stored, and must not send their warp down the masked path
        const int hi_key = live ? pos + 1 : 1 << 30, lo_key = live && a.window > 0 ? max(0, pos + 1 - a.window) : 0;
        const int64_t row0 = it.rr.start + t0;  // the tile's first token
        uint8_t* tile = sm + x * KT_TILE;       // its queries, and at the end its output
        float qs = 0.f, qb = 0.f;
        if (b0 < b1) {
            // The row to shared memory as fp16 (bf16: times a power of two, as in kv8_attn.cu), and its sum. The loads take
            // two rows at a time (a row per thread would touch 32 lines with each of them), so the rows go through
            // shared memory on their way to their threads, too.
            uint32_t w[64];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int row = (warp & 3) * 32 + 2 * i + (lane >> 4), tk = token_of(row);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (tk < nt)
                    v = *(const uint4*)((const T*)a.q.in + (row0 + tk) * a.q.in_token + (int64_t)(kvh * group + row - tk * group) * a.q.in_head +
                                        8 * (lane & 15));
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 16; i++)
                *(uint4*)(tile + tile_off((warp & 3) * 32 + 2 * i + (lane >> 4), lane & 15)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < 16; c++) {
                const uint4 v = *(const uint4*)(tile + tile_off(r, c));
                w[4 * c] = v.x, w[4 * c + 1] = v.y, w[4 * c + 2] = v.z, w[4 * c + 3] = v.w;
            }
            float f = 1.f;
            if (std::is_same<T, __nv_bfloat16>::value) {
                float amax = 0.f;
#pragma unroll
                for (int e = 0; e < 64; e++)
                    amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
                const int ex = min(max((int)((__float_as_uint(amax) >> 23) & 0xff), 14), 254);
                const float up = __uint_as_float((uint32_t)(267 - ex) << 23);
                f = 1.f / up;
#pragma unroll
                for (int e = 0; e < 64; e++) {
                    const __half2 h = __floats2half2_rn(__uint_as_float(w[e] << 16) * up, __uint_as_float(w[e] & 0xffff0000u) * up);
                    w[e] = *(const uint32_t*)&h;
                }
            }
            // a negative scale is taken into the row, so that the keys' factors below are never negative
            f *= fabsf(a.scale);
            const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 64; e++) {
                w[e] ^= sign;
                const float2 h = __half22float2(*(const __half2*)&w[e]);
                sum += h.x + h.y;
            }
            qs = f * 16777216.f;  // K is there as (b + 128) 2^-24
            qb = -128.f * sum * f;
#pragma unroll
            for (int c = 0; c < 16; c++)
                *(uint4*)(tile + tile_off(r, c)) = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + 8 * x);
        }
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_col = tmem + lanes + (uint32_t)(x * 128), s_col = tmem + lanes + 256u + (uint32_t)(x * 128);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int b = b0; b < b1; b++) {
            if (!warp_wait(s_full + 8 * x, (uint32_t)((b - b0) & 1))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const float4* sc = scales + ((b - it.lo) & (KT_SLOTS - 1)) * 8;
            const int k0 = b * KT_KEYS, vis_hi = hi_key - k0, vis_lo = lo_key - k0;
            const bool all = __all_sync(0xffffffffu, vis_hi >= KT_KEYS && vis_lo <= 0);
            // The block in two halves of 64 keys, so that a thread holds 64 scores and not 128.
            uint32_t v[64];
            auto load = [&](int half) {
                uint32_t(&v0)[32] = *reinterpret_cast<uint32_t(*)[32]>(&v[0]);
                uint32_t(&v1)[32] = *reinterpret_cast<uint32_t(*)[32]>(&v[32]);
                tld32(s_col + (uint32_t)(64 * half), v0);
                tld32(s_col + (uint32_t)(64 * half + 32), v1);
                tld_wait(v0);
                tld_wait(v1);
            };
            // The half's largest exponent. Where some row does not see the whole block, v becomes the exponents
            // themselves, masked.
            auto largest = [&](int half) {
                float bm = -INFINITY;
                if (!all) {
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const float4 s = sc[4 * half + h];
                        const float ka = s.x * qs, kb = fmaf(s.x, qb, s.y);
#pragma unroll
                        for (int e = 16 * h; e < 16 * h + 16; e++) {
                            const float y = fmaf(__uint_as_float(v[e]), ka, kb);
                            v[e] = __float_as_uint(64 * half + e < vis_hi && 64 * half + e >= vis_lo ? y : -INFINITY);
                            bm = fmaxf(bm, __uint_as_float(v[e]));
                        }
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const float4 s = sc[4 * half + h];
                        // three inputs at a time, in two chains
                        float g = max3(__uint_as_float(v[16 * h]), __uint_as_float(v[16 * h + 1]), __uint_as_float(v[16 * h + 2]));
                        float g1 = max3(__uint_as_float(v[16 * h + 3]), __uint_as_float(v[16 * h + 4]), __uint_as_float(v[16 * h + 5]));
#pragma unroll
                        for (int e = 16 * h + 6; e < 16 * h + 14; e += 4) {
                            g = max3(g, __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
                            g1 = max3(g1, __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
                        }
                        g = max3(fmaxf(g, g1), __uint_as_float(v[16 * h + 14]), __uint_as_float(v[16 * h + 15]));
                        bm = fmaxf(bm, fmaf(g, s.x * qs, fmaf(s.x, qb, s.y)));
                    }
                }
                return bm;
            };
            // The half's weights as fp16 pairs in v[0..31], and their sum over the values' scales.
            auto weights = [&](int half, float ref) {
                float rs = 0.f;
#pragma unroll
                for (int h = 0; h < 4; h++) {
                    const float4 s = sc[4 * half + h];
                    const float ka = all ? s.x * qs : 1.f, kb = (all ? fmaf(s.x, qb, s.y) : 0.f) - ref;
                    const uint64_t ka2 = pack_f32x2(ka, ka), kb2 = pack_f32x2(kb, kb);
                    uint64_t g2 = 0;
#pragma unroll
                    for (int e = 16 * h; e < 16 * h + 16; e += 2) {
                        const float2 y = unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), ka2, kb2));
                        const float w0 = ex2(y.x), w1 = ex2(y.y);
                        g2 = add_f32x2(g2, pack_f32x2(w0, w1));
                        const __half2 hp = __floats2half2_rn(w0, w1);
                        v[e >> 1] = *reinterpret_cast<const uint32_t*>(&hp);
                    }
                    const float2 gs = unpack_f32x2(g2);
                    rs = fmaf(gs.x + gs.y, s.z, rs);
                }
                return rs;
            };
            auto store = [&](int half) {
#pragma unroll
                for (int c = 0; c < 8; c++)
                    *(uint4*)(sm + (5 + x) * KT_TILE + tile_off(r, 8 * half + c)) = make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
            };
            load(0);
            float bm = largest(0);
            float mn = bm > m + 8.f ? bm : m;
            float rs = weights(0, mn == -INFINITY ? 0.f : mn);
            // W is free, and O holds every block before b, once W V(b - 1) is done
            if (b > b0 && !warp_wait(o_done + 8 * x, (uint32_t)((b - 1 - b0) & 1))) {
                ok = false;
                break;
            }
            tc_fence_after();
            store(0);
            load(1);
            bm = largest(1);
            if (__any_sync(0xffffffffu, bm > mn + 8.f)) {
                // the second half moves a row's reference: the first again, at the new one
                mn = bm > mn + 8.f ? bm : mn;
                load(0);
                largest(0);
                rs = weights(0, mn == -INFINITY ? 0.f : mn);
                store(0);
                load(1);
                largest(1);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_free + 8 * x);  // S(b + 1) may overwrite S(b)
            rs += weights(1, mn == -INFINITY ? 0.f : mn);
            store(1);
            const float alpha = mn == m ? 1.f : m == -INFINITY ? 0.f : ex2(m - mn);
            l = fmaf(l, alpha, rs);
            m = mn;
            // O *= alpha where a row's reference moved
            if (b > b0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                for (int h = 0; h < 4; h++) {
                    uint32_t o[32];
                    tld32(o_col + (uint32_t)(h * 32), o);
                    tld_wait(o);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                    tst32(o_col + (uint32_t)(h * 32), o);
                }
            }
            tst_wait();
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * x);
        }
        const bool any = b0 < b1;
        if (ok && any) ok = warp_wait(o_done + 8 * x, (uint32_t)((b1 - 1 - b0) & 1));
        if (!ok) {
            if (lane == 0) paged_report(err, JV_ERR_DEVICE_TIMEOUT, PS_ATTN_TC + KR_SOFTMAX);
        } else {
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
            __half2 most = __floats2half2_rn(0.f, 0.f);  // the row's largest fp16 outputs: infinities and NaN stay
            const int64_t part = ((int64_t)place * kvh_n + kvh) * 2 * PG_TILE + x * PG_TILE + r;
            // the rows through shared memory (the queries' tile is free now), so that a store takes whole lines
#pragma unroll 1
            for (int h = 0; h < 4; h++) {
                uint32_t o[32];
                if (any) {
                    tld32(o_col + (uint32_t)(h * 32), o);
                    tld_wait(o);
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = 0;
                }
                if (splits == 1) {
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        uint32_t y[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float y0 = __uint_as_float(o[8 * c + 2 * e]) * inv, y1 = __uint_as_float(o[8 * c + 2 * e + 1]) * inv;
                            if (std::is_same<T, __half>::value) {
                                const __half2 q = __floats2half2_rn(y0, y1);
                                most = __hmax2_nan(most, __habs2(q));
                                y[e] = *(const uint32_t*)&q;
                            } else {
                                const __nv_bfloat162 q = __floats2bfloat162_rn(y0, y1);
                                y[e] = *(const uint32_t*)&q;
                            }
                        }
                        *(uint4*)(tile + tile_off(r, 4 * h + c)) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                } else if (any) {  // without a block, the reference of -infinity below says so
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        *(uint4*)(tile + tile_off(r, c)) = make_uint4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int row = (warp & 3) * 32 + 4 * i + (lane >> 3);
                        if (token_of(row) < nt)
                            *(uint4*)(a.large_o + (part - r + row) * PG_DIM + 32 * h + 4 * (lane & 7)) = *(const uint4*)(tile + tile_off(row, lane & 7));
                    }
                    __syncwarp();
                }
            }
            if (splits == 1) {
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int row = (warp & 3) * 32 + 2 * i + (lane >> 4), tk = token_of(row);
                    if (tk < nt)
                        *(uint4*)((T*)a.q.out + (row0 + tk) * a.q.out_token + (int64_t)(kvh * group + row - tk * group) * a.q.out_head + 8 * (lane & 15)) =
                            *(const uint4*)(tile + tile_off(row, lane & 15));
                }
            }
            if (live && !(__half2float(__hmax_nan(__low2half(most), __high2half(most))) < 65520.f)) paged_report(err, JV_ERR_NUMERIC, PS_ATTN_VALUE);
            if (live && splits > 1) a.large_ml[part] = make_float2(m, l);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the splits of pairs of tiles: the grid's warps find the pairs that have some, 32 items a look, and
// take a row each.
constexpr int KTJ_WARPS = 8;
template <class T>
__device__ __forceinline__ bool join_row(const AttnKArgs& a, int4 item, int kvh, int row, int lane) {
    const int splits = item.w & 255, place = item.w >> 8;
    RequestRows rr;
    if (splits > PG_SPLIT_ITEMS || place < 0 || place + splits > a.v.split_cap || !request_rows(a.b, item.x, rr)) return false;
    const int group = a.b.group, tt = PG_TILE / group, x = row / PG_TILE, r = row % PG_TILE, tok = r / group;
    const int t = item.y * 2 * tt + x * tt + tok;
    if (tok >= tt || t < 0 || t >= rr.n_new) return false;
    const int64_t p0 = ((int64_t)place * a.c.kv_heads + kvh) * 2 * PG_TILE + row, step = (int64_t)a.c.kv_heads * 2 * PG_TILE;
    const float2 ml = lane < splits ? a.large_ml[p0 + lane * step] : make_float2(-INFINITY, 0.f);  // at most 16 splits
    float m = ml.x;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float f = ex2(ml.x - (m == -INFINITY ? 0.f : m));
    float l = ml.y * f;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < splits; s++) {
        const float g = __shfl_sync(0xffffffffu, f, s);
        if (g == 0.f) continue;  // also the splits without a block, which left no values
        const float4 y = *(const float4*)(a.large_o + (p0 + s * step) * PG_DIM + 4 * lane);
        o.x = fmaf(y.x, g, o.x), o.y = fmaf(y.y, g, o.y), o.z = fmaf(y.z, g, o.z), o.w = fmaf(y.w, g, o.w);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = (T*)a.q.out + (int64_t)(rr.start + t) * a.q.out_token + (int64_t)(kvh * group + r - tok * group) * a.q.out_head + 4 * lane;
    o.x *= inv, o.y *= inv, o.z *= inv, o.w *= inv;
    if (std::is_same<T, __half>::value) {
        const __half2 u = __floats2half2_rn(o.x, o.y), v = __floats2half2_rn(o.z, o.w);
        *(uint2*)dst = make_uint2(*(const uint32_t*)&u, *(const uint32_t*)&v);
    } else {
        const __nv_bfloat162 u = __floats2bfloat162_rn(o.x, o.y), v = __floats2bfloat162_rn(o.z, o.w);
        *(uint2*)dst = make_uint2(*(const uint32_t*)&u, *(const uint32_t*)&v);
    }
    return outside<T>(o);
}
template <class T>
__global__ void __launch_bounds__(KTJ_WARPS * 32) k_kv8_large_join(AttnKArgs a) {
    pdl_wait();
    bool out_of_range = false;
    const int lane = threadIdx.x & 31, warp = blockIdx.x * KTJ_WARPS + (threadIdx.x >> 5), warps = gridDim.x * KTJ_WARPS;
    const int n = (int)min((int64_t)a.v.head[1], a.v.large_cap);
    for (int i0 = 0; i0 < n; i0 += 32) {
        const int4 mine = i0 + lane < n ? a.v.large_items[i0 + lane] : make_int4(0, 0, 1, 0);
        uint32_t some = __ballot_sync(0xffffffffu, mine.z == 0 && (mine.w & 255) > 1);
        for (; some; some &= some - 1) {
            const int src = __ffs(some) - 1;
            const int4 item = make_int4(__shfl_sync(0xffffffffu, mine.x, src), __shfl_sync(0xffffffffu, mine.y, src),
                                        __shfl_sync(0xffffffffu, mine.z, src), __shfl_sync(0xffffffffu, mine.w, src));
            for (int u = warp; u < a.c.kv_heads * 2 * PG_TILE; u += warps)
                out_of_range |= join_row<T>(a, item, u / (2 * PG_TILE), u % (2 * PG_TILE), lane);
        }
    }
    if (out_of_range) paged_report(a.b.status, JV_ERR_NUMERIC, PS_ATTN_VALUE);
}

template <class T>
void launch_large(const AttnKArgs& a, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    JV_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (!(done.load() & bit)) {
        JV_CUDA(cudaFuncSetAttribute(k_kv8_large<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, KT_SMEM));
        // the softmax's registers come out of what the launch was given: a build with fewer would wait for them for good
        cudaFuncAttributes at;
        JV_CUDA(cudaFuncGetAttributes(&at, k_kv8_large<T>));
        if (at.numRegs != 128) throw Error(JV_ERR_DEVICE, "k_kv8_large was not built with 128 registers per thread");
        done.fetch_or(bit);
    }
    const unsigned items = (unsigned)(a.v.large_cap * a.c.kv_heads);  // jv_kv8_attention has seen that it fits
    launch_pdl(k_kv8_large<T>, dim3(items), dim3(KT_THREADS), KT_SMEM, s, a);
    note_launch();
    if (a.v.split_cap > 0 && a.b.max_blocks > 16) {  // a request of at most 1024 keys has no splits
        launch_pdl(k_kv8_large_join<T>, dim3(2 * 148), dim3(KTJ_WARPS * 32), 0, s, a);
        note_launch();
    }
}

}  // namespace

void launch_kv8_large(const AttnKArgs& a, int type, cudaStream_t s) {
    if (type == T_F16)
        launch_large<__half>(a, s);
    else
        launch_large<__nv_bfloat16>(a, s);
}

}  // namespace jv
