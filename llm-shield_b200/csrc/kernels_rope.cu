// kernels_rope.cu — rotary positions on device buffers (jv_rope) and the write of new keys and
// values into the 8-bit paged cache, rotated on the way (jv_kv8_append).
//
// The rotation of a pair (a, b) at position p: (a cos t - b sin t, a sin t + b cos t) * mscale with
// t = p * freq. p * freq is formed in turns in 64 bits and reduced to one turn before it is rounded to
// fp32 (an error of 2^-25 of a half turn at any position), then sincospif. A CTA computes the angles
// of its tokens once into shared memory and applies them to all its heads.
#include <cmath>
#include <string>

#include <cuda_bf16.h>

#include "paged.h"

namespace jv {
namespace {

constexpr int RP_THREADS = 256;

__device__ __forceinline__ float2 rope_angle(double turns, int pos, float mscale) {
    double t = turns * (double)pos;
    t -= rint(t);
    float s, c;
    sincospif(2.f * (float)t, &s, &c);
    return make_float2(c * mscale, s * mscale);
}

// The query temperature; a position below 0 has none.
__device__ __forceinline__ float temperature_at(const jv_rope_spec& s, int pos) {
    return pos < 0 ? 1.f : rope_temperature(pos, s.temperature_ctx, s.temperature_scale);
}

template <class T>
__device__ __forceinline__ float ld1(const T* p);
template <>
__device__ __forceinline__ float ld1<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float ld1<__half>(const __half* p) { return __half2float(*p); }
template <>
__device__ __forceinline__ float ld1<__nv_bfloat16>(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void st1(float* p, float v) { *p = v; }
__device__ __forceinline__ void st1(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void st1(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Four consecutive elements; one vector access when `vec` (the caller checked the alignment).
__device__ __forceinline__ void get4(uint2 v, const __half*, float (&x)[4]) {
    const float2 a = __half22float2(*(const __half2*)&v.x), b = __half22float2(*(const __half2*)&v.y);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void get4(uint2 v, const __nv_bfloat16*, float (&x)[4]) {
    x[0] = __uint_as_float(v.x << 16), x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16), x[3] = __uint_as_float(v.y & 0xffff0000u);
}
__device__ __forceinline__ void st4(float* p, bool vec, const float (&x)[4]) {
    if (vec) {
        *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = x[e];
    }
}
__device__ __forceinline__ void st4(__half* p, bool vec, const float (&x)[4]) {
    if (vec) {
        __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        *(uint2*)p = make_uint2(*(uint32_t*)&a, *(uint32_t*)&b);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = __float2half_rn(x[e]);
    }
}
__device__ __forceinline__ void st4(__nv_bfloat16* p, bool vec, const float (&x)[4]) {
    if (vec) {
        __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        *(uint2*)p = make_uint2(*(uint32_t*)&a, *(uint32_t*)&b);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = __float2bfloat16_rn(x[e]);
    }
}

// Four elements as they are in memory, so that many rows can be in flight before the first is converted.
template <class T>
struct Quad {
    uint2 raw;
    __device__ __forceinline__ void load(const T* p, bool vec) {
        if (vec) {
            raw = *(const uint2*)p;
        } else {
            const uint16_t* h = (const uint16_t*)p;
            raw = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
        }
    }
    __device__ __forceinline__ void get(float (&x)[4]) const { get4(raw, (const T*)nullptr, x); }
};
template <>
struct Quad<float> {
    float4 raw;
    __device__ __forceinline__ void load(const float* p, bool vec) {
        raw = vec ? *(const float4*)p : make_float4(p[0], p[1], p[2], p[3]);
    }
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = raw.x, x[1] = raw.y, x[2] = raw.z, x[3] = raw.w; }
};

// ------------------------------------------------------------ rope

struct RopeKArgs {
    jv_rope_spec spec;
    jv_heads x[2];
    const int32_t* positions;
    int tokens, dim, n_heads;  // n_heads: of both operands
};

constexpr int RP_TOKENS = 8;  // tokens per CTA

// One CTA: up to 8 tokens, the heads [blockIdx.y * per_cta, + per_cta) of both operands. A thread
// takes one pair of one head at a time (any layout, stride and alignment).
template <class T>
__global__ void __launch_bounds__(RP_THREADS) k_rope(RopeKArgs a, int per_cta) {
    __shared__ float2 cs[RP_TOKENS][128];
    __shared__ float temp[RP_TOKENS];
    pdl_wait();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * RP_TOKENS, nt = min(RP_TOKENS, a.tokens - t0);
    const int half = a.spec.rotary_dim >> 1;
    for (int i = threadIdx.x; i < nt * half; i += RP_THREADS) {
        const int t = i / half, f = i % half;
        cs[t][f] = rope_angle(a.spec.turns[f], a.positions[t0 + t], a.spec.mscale);
    }
    if (threadIdx.x < nt)
        temp[threadIdx.x] = temperature_at(a.spec, a.positions[t0 + threadIdx.x]);
    __syncthreads();
    const int h0 = blockIdx.y * per_cta, nh = min(per_cta, a.n_heads - h0), pairs = a.dim >> 1;
    for (int i = threadIdx.x; i < nt * nh * pairs; i += RP_THREADS) {
        const int p = i % pairs, th = i / pairs, h = h0 + th % nh, t = th / nh;
        const bool second = h >= a.x[0].heads;
        const jv_heads& x = a.x[second ? 1 : 0];
        const int hh = second ? h - a.x[0].heads : h;
        const T* in = (const T*)x.in + (int64_t)(t0 + t) * x.in_token + (int64_t)hh * x.in_head;
        T* out = (T*)x.out + (int64_t)(t0 + t) * x.out_token + (int64_t)hh * x.out_head;
        const float k = x.temperature ? temp[t] : 1.f;
        int e0 = 2 * p, e1 = 2 * p + 1;
        if (p < half && a.spec.layout == JV_ROPE_HALF) e0 = p, e1 = p + half;
        float u = ld1(in + e0), v = ld1(in + e1);
        if (p < half) {
            const float2 c = cs[t][p];
            const float r = fmaf(-v, c.y, u * c.x);  // as rotate_vec has it: alignment changes no bits
            v = fmaf(u, c.y, v * c.x);
            u = r;
        }
        st1(out + e0, u * k);
        st1(out + e1, v * k);
    }
}

// The same with 16-byte accesses (V elements), for rows and pair halves that start on 16 bytes. A
// "piece" is V consecutive elements of adjacent pairs, or both halves of V half-split pairs, or, in a second
// sweep, V elements behind rotary_dim; a power of two of lanes takes a head's pieces, so that every lane of a
// warp has the same kind. Bound by HBM: four (token, head) rows per thread in flight, the first four before
// the angles are worked out. 8191 tokens x 40 heads of 128 in bf16, half of each turned: 35 us, 74 % of the
// measured copy rate.
template <class T>
union Vec {
    uint4 raw;
    T e[16 / sizeof(T)];
};
__device__ __forceinline__ void rotate_vec(Vec<float>& u, Vec<float>& v, const float2* cs, bool half_split, float k) {
#pragma unroll
    for (int e = 0; e < 4; e += half_split ? 1 : 2) {
        float& pa = u.e[e];
        float& pb = half_split ? v.e[e] : u.e[e + 1];
        const float2 c = cs[half_split ? e : e >> 1];
        const float x = pa, y = pb;
        pa = fmaf(-y, c.y, x * c.x) * k;
        pb = fmaf(x, c.y, y * c.x) * k;
    }
}
// 16-bit elements, two at a time: (u0, u1) and (v0, v1) of half-split pairs, (u0, u1) a pair itself otherwise.
template <class T>
__device__ __forceinline__ void rotate_vec(Vec<T>& u, Vec<T>& v, const float2* cs, bool half_split, float k) {
    uint32_t* pu = (uint32_t*)&u.raw;
    uint32_t* pv = (uint32_t*)&v.raw;
#pragma unroll
    for (int w = 0; w < 4; w += 2) {
        float x[4], y[4];
        get4(make_uint2(pu[w], pu[w + 1]), (const T*)nullptr, x);
        if (half_split) {
            get4(make_uint2(pv[w], pv[w + 1]), (const T*)nullptr, y);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 c = cs[2 * w + e];
                const float r = fmaf(-y[e], c.y, x[e] * c.x);
                y[e] = fmaf(x[e], c.y, y[e] * c.x);
                x[e] = r;
            }
            if (k != 1.f)
                for (int e = 0; e < 4; e++) y[e] *= k;
            st4((T*)(pv + w), true, y);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float2 c = cs[w + e / 2];
                const float r = fmaf(-x[e + 1], c.y, x[e] * c.x);
                x[e + 1] = fmaf(x[e], c.y, x[e + 1] * c.x);
                x[e] = r;
            }
        }
        if (k != 1.f)
            for (int e = 0; e < 4; e++) x[e] *= k;
        st4((T*)(pu + w), true, x);
    }
}
template <class T>
__device__ __forceinline__ void scale_vec(Vec<T>& u, float k) {
#pragma unroll
    for (int e = 0; e < (int)(16 / sizeof(T)); e++) st1(u.e + e, ld1(u.e + e) * k);
}

template <class T, int LAYOUT>
__global__ void __launch_bounds__(RP_THREADS) k_rope_vec(RopeKArgs a, int per_cta, int turn_bits, int rest_bits) {
    constexpr int V = 16 / sizeof(T), U = 4;
    constexpr bool SPLIT = LAYOUT == JV_ROPE_HALF;
    __shared__ __align__(16) float2 cs[RP_TOKENS][128];
    __shared__ float temp[RP_TOKENS];
    pdl_wait();
    pdl_launch_dependents();
    const int t0 = blockIdx.x * RP_TOKENS, nt = min(RP_TOKENS, a.tokens - t0);
    const int half = a.spec.rotary_dim >> 1;
    const int h0 = blockIdx.y * per_cta, nh = min(per_cta, a.n_heads - h0);
    Vec<T> u[U], v[U];
    T* out[U];
    int tt[U];  // a row's token, 256 added where it takes the query temperature; 255 without a row
    int t, h, dt, dh, e0;
    bool in_range;
    auto begin = [&](int bits, int pieces, int first) {
        const int piece = threadIdx.x & ((1 << bits) - 1), row = threadIdx.x >> bits, step = RP_THREADS >> bits;
        e0 = first + piece * V;
        in_range = piece < pieces;
        t = row / nh, h = row % nh, dt = step / nh, dh = step % nh;
    };
    auto load = [&](bool turn) {
#pragma unroll
        for (int n = 0; n < U; n++) {
            tt[n] = 255;
            if (t < nt && in_range) {
                const bool second = h0 + h >= a.x[0].heads;
                const jv_heads& x = a.x[second ? 1 : 0];
                const int hh = second ? h0 + h - a.x[0].heads : h0 + h;
                const T* in = (const T*)x.in + (int64_t)(t0 + t) * x.in_token + (int64_t)hh * x.in_head + e0;
                out[n] = (T*)x.out + (int64_t)(t0 + t) * x.out_token + (int64_t)hh * x.out_head + e0;
                tt[n] = t | (x.temperature ? 256 : 0);
                u[n].raw = *(const uint4*)in;
                if (SPLIT && turn) v[n].raw = *(const uint4*)(in + half);
            }
            t += dt;
            h += dh;
            if (h >= nh) h -= nh, t++;
        }
    };
    begin(turn_bits, SPLIT ? half / V : 2 * half / V, 0);
    load(true);
    for (int i = threadIdx.x; i < nt * half; i += RP_THREADS) {
        const int ti = i / half, f = i % half;
        cs[ti][f] = rope_angle(a.spec.turns[f], a.positions[t0 + ti], a.spec.mscale);
    }
    if (threadIdx.x < nt)
        temp[threadIdx.x] = temperature_at(a.spec, a.positions[t0 + threadIdx.x]);
    __syncthreads();
    while (tt[0] != 255) {
#pragma unroll
        for (int n = 0; n < U; n++) {
            if (tt[n] == 255) break;
            rotate_vec(u[n], v[n], cs[tt[n] & 255] + (SPLIT ? e0 : e0 >> 1), SPLIT, tt[n] & 256 ? temp[tt[n] & 255] : 1.f);
            *(uint4*)out[n] = u[n].raw;
            if (SPLIT) *(uint4*)(out[n] + half) = v[n].raw;
        }
        load(true);
    }
    if (a.dim == 2 * half) return;
    begin(rest_bits, (a.dim - 2 * half) / V, 2 * half);
    load(false);
    while (tt[0] != 255) {
#pragma unroll
        for (int n = 0; n < U; n++) {
            if (tt[n] == 255) break;
            if (tt[n] & 256) scale_vec(u[n], temp[tt[n] & 255]);
            *(uint4*)out[n] = u[n].raw;
        }
        load(false);
    }
}

// ------------------------------------------------------------ append

struct AppendArgs {
    jv_kv8_cache c;
    jv_paged_batch b;
    PlanView v;
    jv_heads k, vv, q;
    jv_rope_spec spec;
    bool rope;
    int q_heads;                  // 0 without q
};

// Rotates four consecutive dimensions 4 lane .. 4 lane + 3 of a head held by a warp.
__device__ __forceinline__ void rope4(float (&x)[4], const float2* cs, int layout, int half, int lane) {
    if (layout == JV_ROPE_ADJACENT) {
        if (4 * lane < 2 * half) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float2 c = cs[2 * lane + e / 2];
                const float r = __fsub_rn(__fmul_rn(x[e], c.x), __fmul_rn(x[e + 1], c.y));
                x[e + 1] = __fadd_rn(__fmul_rn(x[e], c.y), __fmul_rn(x[e + 1], c.x));
                x[e] = r;
            }
        }
    } else {
        const int off = half >> 2;  // lanes between the two halves of a pair
        const bool lo = lane < off, in = lane < 2 * off;
        const int other = !in ? lane : lo ? lane + off : lane - off;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float y = __shfl_sync(0xffffffffu, x[e], other);
            if (in) {
                const float2 c = cs[4 * (lo ? lane : other) + e];
                x[e] = lo ? __fsub_rn(__fmul_rn(x[e], c.x), __fmul_rn(y, c.y))
                          : __fadd_rn(__fmul_rn(y, c.y), __fmul_rn(x[e], c.x));
            }
        }
    }
}

// The largest magnitude of four values, as the integer that its bits are: not finite from 0x7f800000 on.
__device__ __forceinline__ uint32_t top4(const float (&x)[4]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ void finite4(const float (&x)[4], float& amax) {
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (fabsf(x[e]) < INFINITY) amax = fmaxf(amax, fabsf(x[e]));
}
// A block's scale and what its values are multiplied by, from each lane's largest magnitude and the scale the
// block had. Where a value is not finite (false), `again` takes the largest of the others.
template <class F>
__device__ __forceinline__ bool block_scale(uint32_t top, float had, float& scale, float& inv, F&& again) {
    top = __reduce_max_sync(0xffffffffu, top);
    const bool finite = top < 0x7f800000u;
    float amax = __uint_as_float(top);
    if (!finite) {
        amax = 0.f;
        again(amax);
        amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    }
    if (amax < 7.888609e-31f) amax = 0.f;  // 2^-100: 127 / amax stays finite
    scale = __fdiv_rn(amax, 127.f);
    inv = amax > 0.f ? __fdiv_rn(127.f, amax) : 0.f;
    if (had > scale) {
        scale = had;
        inv = __fdiv_rn(1.f, had);
    }
    return finite;
}
// x inv rounded to a whole number by adding 1.5 2^23 (|x inv| <= 127, or it is clamped): the low byte of the sum
// is the int8. Four of them in a word.
__device__ __forceinline__ uint32_t quantise4(const float (&x)[4], float inv, bool finite) {
    uint32_t q[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float y = __fmul_rn(x[e], inv);
        if (!finite) y = isnan(x[e]) || inv == 0.f ? 0.f : fminf(fmaxf(y, -127.f), 127.f);
        q[e] = __float_as_uint(__fadd_rn(y, 12582912.f));
    }
    return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}

// One CTA: a 16-token block that the step writes to, a slice of its heads; one warp a head at a time
// (a lane holds 4 dimensions of the 16 tokens, so a block's largest magnitude is one register
// reduction over the lanes). Latency-bound: 16 rows of a head are in flight per warp, 16 warps per SM
// (5,500 tokens x 8 KV heads in bf16: 15 us, floor 5.3).
template <class T, class TQ, bool VEC, bool ROPE>
__global__ void __launch_bounds__(RP_THREADS, 2) k_kv8_append(AppendArgs a) {
    __shared__ float2 cs[PG_BLOCK][64];
    __shared__ float temp[PG_BLOCK];
    pdl_wait();
    pdl_launch_dependents();
    if ((int)blockIdx.x >= a.v.head[2]) return;
    const int4 unit = a.v.units[blockIdx.x];
    // rows [lo, hi) of the block are new, token tok0 + row each; [0, lo) are kept
    const int p0 = unit.y * PG_BLOCK, tok0 = unit.z, lo = unit.w & 255, hi = unit.w >> 8;
    if ((unsigned)unit.x >= (unsigned)a.b.requests || (unsigned)unit.y >= (unsigned)a.b.max_blocks * (PG_TOKENS / PG_BLOCK) || lo >= hi ||
        hi > PG_BLOCK || tok0 + lo < 0 || tok0 > a.b.max_tokens - hi)
        return;
    const int page = a.b.block_table[(int64_t)unit.x * a.b.max_blocks + p0 / PG_TOKENS];
    if ((unsigned)page >= (unsigned)a.c.pages) {
        if (threadIdx.x == 0) paged_report(a.b.status, JV_ERR_RANGE, PS_APPEND_PAGE);
        return;
    }
    const int half = a.spec.rotary_dim >> 1;
    if (ROPE) {
        for (int i = threadIdx.x; i < PG_BLOCK * half; i += RP_THREADS) {
            const int t = i / half, f = i % half;
            if (t >= lo && t < hi) cs[t][f] = rope_angle(a.spec.turns[f], p0 + t, a.spec.mscale);
        }
        if (threadIdx.x < PG_BLOCK)
            temp[threadIdx.x] = temperature_at(a.spec, p0 + threadIdx.x);
        __syncthreads();
    }
    const int lane = threadIdx.x & 31, g = a.c.kv_heads;
    const int n_work = 2 * g + a.q_heads;
    for (int w = blockIdx.y * (RP_THREADS / 32) + (threadIdx.x >> 5); w < n_work; w += gridDim.y * (RP_THREADS / 32)) {
        if (ROPE && w >= 2 * g) {  // a query head: rotate and hand on
            const int h = w - 2 * g;
            bool bad = false;
            const T* in = (const T*)a.q.in + (int64_t)tok0 * a.q.in_token + (int64_t)h * a.q.in_head + 4 * lane;
            TQ* out = (TQ*)a.q.out + (int64_t)tok0 * a.q.out_token + (int64_t)h * a.q.out_head + 4 * lane;
            for (int t0 = lo; t0 < hi; t0 += 8) {
                Quad<T> r[8];
#pragma unroll
                for (int t = 0; t < 8; t++)
                    if (t0 + t < hi) r[t].load(in + (t0 + t) * a.q.in_token, VEC);
#pragma unroll
                for (int t = 0; t < 8; t++) {
                    if (t0 + t >= hi) break;
                    float x[4];
                    r[t].get(x);
                    rope4(x, cs[t0 + t], a.spec.layout, half, lane);
                    const float k = a.q.temperature ? temp[t0 + t] : 1.f;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] *= k;
                        if (std::is_same<TQ, __half>::value) bad |= f16_out_of_range(x[e]);
                    }
                    st4(out + (t0 + t) * a.q.out_token, VEC, x);
                }
            }
            if (__any_sync(0xffffffffu, bad) && lane == 0) paged_report(a.b.status, JV_ERR_NUMERIC, PS_ROPE_VALUE);
            continue;
        }
        const int h = w >> 1, kv = w & 1;
        const jv_heads& src = kv ? a.vv : a.k;
        const bool turn = ROPE && kv == 0;
        const T* in = (const T*)src.in + (int64_t)tok0 * src.in_token + (int64_t)h * src.in_head + 4 * lane;
        float* sp = a.c.scales + (int64_t)page * a.c.scale_stride + (h * 2 + kv) * 4 + (p0 % PG_TOKENS) / PG_BLOCK;
        char* dst = (char*)a.c.data + (int64_t)page * a.c.page_bytes + (int64_t)(h * 2 + kv) * PG_PLANE +
                    (p0 % PG_TOKENS) * PG_DIM + 4 * lane;
        float scale;
        if (lo == 0 && hi == PG_BLOCK && !(ROPE && sizeof(T) == 4)) {
            // a whole block: its rows in registers, no entries to keep, no row to leave out (fp32 rows with their
            // angles would not fit: those go four at a time)
            float x[PG_BLOCK][4];
            {
                Quad<T> raw[PG_BLOCK];
#pragma unroll
                for (int t = 0; t < PG_BLOCK; t++) raw[t].load(in + t * src.in_token, VEC);
#pragma unroll
                for (int t = 0; t < PG_BLOCK; t++) raw[t].get(x[t]);
            }
            if (turn) {
#pragma unroll
                for (int t = 0; t < PG_BLOCK; t++) rope4(x[t], cs[t], a.spec.layout, half, lane);
            }
            uint32_t top = 0;
#pragma unroll
            for (int t = 0; t < PG_BLOCK; t++) top = max(top, top4(x[t]));
            float inv;
            const bool finite = block_scale(top, 0.f, scale, inv, [&](float& amax) {
#pragma unroll
                for (int t = 0; t < PG_BLOCK; t++) finite4(x[t], amax);
            });
            if (!finite && lane == 0) paged_report(a.b.status, JV_ERR_NUMERIC, PS_APPEND_VALUE);
#pragma unroll
            for (int t = 0; t < PG_BLOCK; t++) *(uint32_t*)(dst + t * PG_DIM) = quantise4(x[t], inv, finite);
        } else {
            // part of a block: four rows at a time, read twice
            auto rows = [&](auto&& use) {
                for (int t0 = lo; t0 < hi; t0 += 4) {
                    Quad<T> raw[4];
#pragma unroll
                    for (int t = 0; t < 4; t++)
                        if (t0 + t < hi) raw[t].load(in + (t0 + t) * src.in_token, VEC);
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        if (t0 + t >= hi) break;
                        float x[4];
                        raw[t].get(x);
                        if (turn) rope4(x, cs[t0 + t], a.spec.layout, half, lane);
                        use(t0 + t, x);
                    }
                }
            };
            const float had = lo > 0 ? *sp : 0.f;
            uint32_t top = 0;
            rows([&](int, const float (&x)[4]) { top = max(top, top4(x)); });
            float inv;
            const bool finite = block_scale(top, had, scale, inv, [&](float& amax) { rows([&](int, const float (&x)[4]) { finite4(x, amax); }); });
            if (!finite && lane == 0) paged_report(a.b.status, JV_ERR_NUMERIC, PS_APPEND_VALUE);
            // values kept from earlier steps, at the grown scale (an 8-bit value again, off by half a step at most)
            if (lo > 0 && had != scale) {
                const float ratio = scale > 0.f ? __fdiv_rn(had, scale) : 0.f;
#pragma unroll 4
                for (int t = 0; t < lo; t++) {
                    char4 o = *(char4*)(dst + t * PG_DIM);
                    o.x = (signed char)rintf(o.x * ratio);
                    o.y = (signed char)rintf(o.y * ratio);
                    o.z = (signed char)rintf(o.z * ratio);
                    o.w = (signed char)rintf(o.w * ratio);
                    *(char4*)(dst + t * PG_DIM) = o;
                }
            }
            rows([&](int t, const float (&x)[4]) { *(uint32_t*)(dst + t * PG_DIM) = quantise4(x, inv, finite); });
        }
        __syncwarp();
        if (lane == 0) *sp = scale;
    }
}

// ------------------------------------------------------------ host

void check_heads(const jv_heads* x, const char* name, int heads, int elem, bool in, bool out) {
    const std::string n(name);
    if (!x) throw Error(JV_ERR_ARG, n + " is NULL");
    if (heads >= 0 && x->heads != heads) throw Error(JV_ERR_ARG, n + " must have " + std::to_string(heads) + " heads");
    if (x->heads < 1 || x->heads > 16384) throw Error(JV_ERR_ARG, n + " must have 1 to 16384 heads");
    if ((in && !x->in) || (out && !x->out)) throw Error(JV_ERR_ARG, n + " has a NULL buffer");
    if ((in && (uintptr_t)x->in % elem) || (out && elem > 0 && (uintptr_t)x->out % 2))
        throw Error(JV_ERR_ARG, n + " is not aligned to its elements");
    if ((in && (x->in_token < 0 || x->in_head < 0)) || (out && (x->out_token < 0 || x->out_head < 0)))
        throw Error(JV_ERR_ARG, n + " has a negative stride");
}

bool vec4(const void* p, int64_t a, int64_t b, int elem) {
    return (uintptr_t)p % (4 * elem) == 0 && a % 4 == 0 && b % 4 == 0;
}

template <class T>
void launch_rope(const RopeKArgs& a, int n, cudaStream_t s) {
    const int tiles = (a.tokens - 1) / RP_TOKENS + 1;  // tokens is 1 to 2^31 - 1
    // enough CTAs for the SMs when the tokens are few: the heads are split
    const int split = std::max(1, std::min(a.n_heads, 1184 / std::max(1, tiles)));
    const int per = (a.n_heads + split - 1) / split;
    const dim3 grid(tiles, (a.n_heads + per - 1) / per);
    constexpr int V = 16 / sizeof(T);
    const bool half_split = a.spec.layout == JV_ROPE_HALF;
    bool vec = a.dim % V == 0 && a.spec.rotary_dim % (half_split ? 2 * V : V) == 0;
    for (int i = 0; i < n; i++) {
        const jv_heads& x = a.x[i];
        vec = vec && (uintptr_t)x.in % 16 == 0 && (uintptr_t)x.out % 16 == 0 && x.in_token % V == 0 && x.in_head % V == 0 &&
              x.out_token % V == 0 && x.out_head % V == 0;
    }
    if (vec) {
        auto bits = [](int pieces) {
            int b = 0;
            while ((1 << b) < pieces) b++;
            return b;
        };
        const int turn = bits(a.spec.rotary_dim / (half_split ? 2 * V : V)), rest = bits((a.dim - a.spec.rotary_dim) / V);
        if (half_split)
            launch_pdl(k_rope_vec<T, JV_ROPE_HALF>, grid, dim3(RP_THREADS), 0, s, a, per, turn, rest);
        else
            launch_pdl(k_rope_vec<T, JV_ROPE_ADJACENT>, grid, dim3(RP_THREADS), 0, s, a, per, turn, rest);
    } else {
        launch_pdl(k_rope<T>, grid, dim3(RP_THREADS), 0, s, a, per);
    }
    note_launch();
}

template <class T, class TQ>
void launch_append(const AppendArgs& a, bool vec, cudaStream_t s) {
    // A head per warp, unless the angles that every CTA works out would then cost more than its heads: with
    // rope, as many CTAs as fill the SMs.
    const int warps = RP_THREADS / 32, work = 2 * a.c.kv_heads + a.q_heads;
    const int most = (work + warps - 1) / warps;
    const int split = !a.rope ? most : (int)std::max<int64_t>(1, std::min<int64_t>(most, 592 / std::max<int64_t>(1, a.v.unit_cap)));
    const dim3 grid((unsigned)a.v.unit_cap, split);
    auto go = [&](auto kernel) { launch_pdl(kernel, grid, dim3(RP_THREADS), 0, s, a); };
    if (a.rope)
        vec ? go(k_kv8_append<T, TQ, true, true>) : go(k_kv8_append<T, TQ, false, true>);
    else
        vec ? go(k_kv8_append<T, __half, true, false>) : go(k_kv8_append<T, __half, false, false>);
    note_launch();
}

void check_spec(const jv_rope_spec* r) {
    if (!r) throw Error(JV_ERR_ARG, "the rope spec is NULL");
    if (r->layout != JV_ROPE_ADJACENT && r->layout != JV_ROPE_HALF) throw Error(JV_ERR_ARG, "rope: unknown layout");
    if (r->rotary_dim < 2 || r->rotary_dim > 256 || r->rotary_dim % 2) throw Error(JV_ERR_ARG, "rope: rotary_dim must be even, 2 to 256");
    if (r->temperature_ctx < 0) throw Error(JV_ERR_ARG, "rope: temperature_ctx is negative");
}

}  // namespace
}  // namespace jv

using namespace jv;

extern "C" {

int jv_rope_init(jv_rope_spec* out, int32_t layout, int32_t rotary_dim, double base, int32_t scaling, double factor,
                 int32_t original_context, double beta_fast, double beta_slow, double attn_factor) {
    return paged_api([&] {
        if (!out) throw Error(JV_ERR_ARG, "the rope spec is NULL");
        jv_rope_spec r{};
        r.layout = layout;
        r.rotary_dim = rotary_dim;
        check_spec(&r);
        if (!(base > 0) || !std::isfinite(base)) throw Error(JV_ERR_ARG, "rope: base must be positive");
        if (scaling < JV_ROPE_PLAIN || scaling > JV_ROPE_YARN) throw Error(JV_ERR_ARG, "rope: unknown scaling");
        if (scaling != JV_ROPE_PLAIN && (!(factor > 0) || !std::isfinite(factor)))
            throw Error(JV_ERR_ARG, "rope: factor must be positive");
        if (!std::isfinite(attn_factor)) throw Error(JV_ERR_ARG, "rope: attn_factor must be finite");
        const double two_pi = 6.283185307179586476925286766559;
        double low = 0, high = 0, ms = attn_factor;
        if (scaling == JV_ROPE_YARN) {
            if (original_context < 1 || !(beta_fast > 0) || !(beta_slow > 0) || !(base > 1))
                throw Error(JV_ERR_ARG, "rope: YaRN needs original_context, beta_fast, beta_slow and a base above 1");
            auto corr = [&](double rot) { return rotary_dim * std::log(original_context / (rot * two_pi)) / (2 * std::log(base)); };
            low = std::max(0.0, std::floor(corr(beta_fast)));
            high = std::min(rotary_dim / 2.0 - 1.0, std::ceil(corr(beta_slow)));
            if (factor > 1) ms *= 0.1 * std::log(factor) + 1.0;
        }
        r.mscale = (float)ms;
        for (int i = 0; i < rotary_dim / 2; i++) {
            double f = std::pow(base, -2.0 * i / rotary_dim);
            if (scaling == JV_ROPE_LINEAR) f /= factor;
            if (scaling == JV_ROPE_YARN) {
                const double y = (i - low) / std::max(0.001, high - low);
                const double keep = 1.0 - std::min(std::max(y, 0.0), 1.0);
                f = f / factor * (1 - keep) + f * keep;
            }
            r.turns[i] = f / two_pi;
        }
        *out = r;
    });
}

int jv_rope(const jv_rope_spec* spec, int32_t type, const int32_t* positions, int32_t tokens, int32_t head_dim,
            const jv_heads* x, int32_t n, void* stream) {
    return paged_api([&] {
        check_spec(spec);
        const int elem = type_bytes(type);
        if (elem == 0) throw Error(JV_ERR_UNSUPPORTED, "the type must be F32 (0), F16 (1) or BF16 (30)");
        if (head_dim < 2 || head_dim > 256 || head_dim % 2) throw Error(JV_ERR_ARG, "rope: head_dim must be even, 2 to 256");
        if (spec->rotary_dim > head_dim) throw Error(JV_ERR_ARG, "rope: rotary_dim is larger than head_dim");
        if (n < 1 || n > 2 || !x) throw Error(JV_ERR_ARG, "rope: one or two operands");
        if (tokens < 0) throw Error(JV_ERR_ARG, "rope: tokens is negative");
        RopeKArgs a{};
        a.n_heads = 0;
        for (int i = 0; i < n; i++) {
            check_heads(x + i, i ? "the second operand" : "the first operand", -1, elem, true, true);
            if ((uintptr_t)x[i].out % elem) throw Error(JV_ERR_ARG, "rope: an output is not aligned to its elements");
            check_rows(x + i, "rope", head_dim, tokens);
            if (x[i].in == x[i].out && ((x[i].in_token != x[i].out_token && tokens > 1) || (x[i].in_head != x[i].out_head && x[i].heads > 1)))
                throw Error(JV_ERR_ARG, "rope: an operand in place must have the same strides in and out");
            a.x[i] = x[i];
            a.n_heads += x[i].heads;
        }
        if (tokens == 0) return;
        if (!positions) throw Error(JV_ERR_ARG, "NULL buffer");
        OnDeviceOf dev(x[0].out);
        a.spec = *spec;
        a.positions = positions;
        a.tokens = tokens;
        a.dim = head_dim;
        cudaStream_t s = (cudaStream_t)stream;
        if (type == T_F32)
            launch_rope<float>(a, n, s);
        else if (type == T_F16)
            launch_rope<__half>(a, n, s);
        else
            launch_rope<__nv_bfloat16>(a, n, s);
    });
}

int jv_kv8_append(const jv_kv8_cache* cache, const jv_paged_batch* batch, int32_t type, const jv_heads* k,
                  const jv_heads* v, const jv_rope_spec* rope, const jv_heads* q, int32_t out_type, void* stream) {
    return paged_api([&] {
        check_cache(cache);
        check_batch(batch, true);
        if (batch->pages != cache->pages) throw Error(JV_ERR_ARG, "the batch and the cache have different numbers of pages");
        const int elem = type_bytes(type);
        if (elem == 0) throw Error(JV_ERR_UNSUPPORTED, "the type must be F32 (0), F16 (1) or BF16 (30)");
        check_heads(k, "k", cache->kv_heads, elem, true, false);
        check_heads(v, "v", cache->kv_heads, elem, true, false);
        if (k->temperature || v->temperature) throw Error(JV_ERR_ARG, "the query temperature is for q, not for k or v");
        AppendArgs a{};
        a.c = *cache;
        a.b = *batch;
        a.v = plan_view(*batch);
        a.k = *k;
        a.vv = *v;
        // four elements at once, where every operand's rows allow it
        bool vec = vec4(k->in, k->in_token, k->in_head, elem) && vec4(v->in, v->in_token, v->in_head, elem);
        a.rope = rope != nullptr;
        if (rope) {
            check_spec(rope);
            if (rope->rotary_dim > PG_DIM || rope->rotary_dim % 8)
                throw Error(JV_ERR_UNSUPPORTED, "rope on the way into the cache needs a rotary_dim that is a multiple of 8, at most 128");
            a.spec = *rope;
        } else {
            a.spec.rotary_dim = 2;
        }
        int oelem = 2;
        if (q) {
            if (!rope) throw Error(JV_ERR_ARG, "q is only taken together with rope");
            oelem = type_bytes(out_type);
            if (oelem == 0) throw Error(JV_ERR_UNSUPPORTED, "the output type must be F32 (0), F16 (1) or BF16 (30)");
            check_heads(q, "q", cache->kv_heads * batch->group, elem, true, true);
            if ((uintptr_t)q->out % oelem) throw Error(JV_ERR_ARG, "q is not aligned to its elements");
            check_rows(q, "q", PG_DIM, 1);  // within a token: max_tokens is only a bound
            if (q->in == q->out && (type != out_type || q->in_token != q->out_token || q->in_head != q->out_head))
                throw Error(JV_ERR_ARG, "q in place must have the same type and strides in and out");
            a.q = *q;
            a.q_heads = q->heads;
            vec = vec && vec4(q->in, q->in_token, q->in_head, elem) && vec4(q->out, q->out_token, q->out_head, oelem);
        }
        OnDeviceOf dev(cache->data);
        cudaStream_t s = (cudaStream_t)stream;
        auto go = [&](auto t) {
            using T = decltype(t);
            if (!q || out_type == T_F16)
                launch_append<T, __half>(a, vec, s);
            else if (out_type == T_F32)
                launch_append<T, float>(a, vec, s);
            else
                launch_append<T, __nv_bfloat16>(a, vec, s);
        };
        if (type == T_F32)
            go(float{});
        else if (type == T_F16)
            go(__half{});
        else
            go(__nv_bfloat16{});
    });
}

}  // extern "C"
