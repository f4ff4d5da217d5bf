// paged.cu — the paged-batch section of include/jv.h: argument checks, the plan of a step (block
// tables, slot maps and work lists built on the GPU from the requests' lengths) and the read-back
// of cache slots.
#include <cmath>
#include <string>

#include <cuda_bf16.h>

#include "paged.h"

namespace jv {

// ------------------------------------------------------------ host checks

int type_bytes(int type) { return type == T_F32 ? 4 : type == T_F16 || type == T_BF16 ? 2 : 0; }

static void need(bool ok, const char* what) {
    if (!ok) throw Error(JV_ERR_ARG, what);
}
static bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

void check_batch(const jv_paged_batch* b, bool arrays) {
    need(b != nullptr, "the batch is NULL");
    need(b->requests >= 1 && b->requests <= PG_MAX_REQUESTS, "a batch has 1 to 4096 requests");
    need(b->max_new >= 1 && b->max_tokens >= 1, "max_new and max_tokens must be at least 1");
    need(b->max_blocks >= 1 && b->max_blocks <= (1 << 24), "max_blocks must be 1 to 2^24");
    need(b->max_tokens <= (1 << 28), "max_tokens must be at most 2^28");
    need(b->max_keys >= 0 && b->max_keys <= (int64_t)b->requests * b->max_blocks * PG_TOKENS,
         "max_keys must be at most requests * max_blocks * 64");
    need(b->group >= 1 && b->group <= PG_MAX_GROUP, "group must be 1 to 16 query heads per KV head");
    need(b->pages >= 1, "the cache needs at least one page");
    if (!arrays) return;
    need(b->block_table && b->lengths && b->starts && b->request_of && b->positions && b->slots && b->work && b->status,
         "a batch array is NULL");
    need(aligned(b->work, 16) && aligned(b->slots, 8) && aligned(b->block_table, 4) && aligned(b->lengths, 4) &&
             aligned(b->starts, 4) && aligned(b->request_of, 4) && aligned(b->positions, 4) && aligned(b->status, 4),
         "a batch array is not aligned");
}

void check_cache(const jv_kv8_cache* c) {
    need(c != nullptr, "the cache is NULL");
    need(c->data && c->scales, "a cache buffer is NULL");
    need(c->pages >= 1 && c->kv_heads >= 1 && c->kv_heads <= 1024, "a cache has at least one page and 1 to 1024 KV heads");
    need(c->page_bytes >= (int64_t)c->kv_heads * 2 * PG_PLANE && c->page_bytes % 16 == 0,
         "page_bytes must be a multiple of 16 and at least kv_heads * 16384");
    need(c->scale_stride >= (int64_t)c->kv_heads * 8 && c->scale_stride % 4 == 0,
         "scale_stride must be a multiple of 4 and at least kv_heads * 8");
    need(aligned(c->data, 16) && aligned(c->scales, 16), "the cache buffers must be 16-byte aligned");
}

// Rows of an output must not lie on one another.
void check_rows(const jv_heads* x, const char* name, int dim, int64_t tokens) {
    const int64_t H = x->heads, a = x->out_token, b = x->out_head;
    const bool token_major = b >= dim && (tokens <= 1 || a >= (H - 1) * b + dim);
    const bool head_major = (tokens <= 1 || a >= dim) && (H <= 1 || b >= (tokens - 1) * a + dim);
    if (!(H == 1 && (tokens <= 1 || a >= dim)) && !token_major && !head_major)
        throw Error(JV_ERR_ARG, std::string(name) + ": rows of the output overlap");
}

OnDeviceOf::OnDeviceOf(const void* p) {
    cudaPointerAttributes at;
    JV_CUDA(cudaPointerGetAttributes(&at, p));
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
        throw Error(JV_ERR_ARG, "the operators of paged batches take device memory");
    int cur = 0;
    JV_CUDA(cudaGetDevice(&cur));
    if (cur != at.device) {
        JV_CUDA(cudaSetDevice(at.device));
        before = cur;
    }
}
OnDeviceOf::~OnDeviceOf() {
    if (before >= 0) cudaSetDevice(before);
}

// ------------------------------------------------------------ plan

PlanView plan_view(const jv_paged_batch& b) {
    PlanView v;
    const int64_t R = b.requests, T = b.max_tokens;
    // small items: a chunk has at least 256 keys except a request's last; units: every one holds a
    // new token, and a request's span has at most new / 16 + 2 of them
    v.small_cap = R + b.max_keys / 256;
    v.large_cap = std::min<int64_t>(R, T * b.group / (PG_SMALL_ROWS + 1)) + T * b.group / PG_TILE_ROWS;
    v.unit_cap = std::min<int64_t>(T, T / PG_BLOCK + 2 * R);
    uint8_t* p = (uint8_t*)b.work;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        uint8_t* r = p ? p + at : nullptr;
        at += (bytes + 15) & ~(int64_t)15;
        return r;
    };
    v.head = (int32_t*)take(8 * 4);
    v.first = (int32_t*)take(R * 4);
    v.prefix = (int32_t*)take(4 * (R + 1) * 4);
    v.small_items = (int4*)take(v.small_cap * 16);
    v.large_items = (int4*)take(v.large_cap * 16);
    v.units = (int2*)take(v.unit_cap * 8);
    v.bytes = at;
    return v;
}

namespace {

struct PlanArgs {
    jv_paged_batch b;
    PlanView v;
    const int32_t* cached;
    const int32_t* new_tokens;
    const int32_t* free_pages;
    const int32_t* n_free;
    int32_t* n_free_out;
};

constexpr int PLAN_THREADS = 1024;

// Exclusive sums over the block of five counts per thread; totals in tot.
__device__ __forceinline__ void block_scan5(int (&x)[5], int (&tot)[5], int (*ws)[5]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc[5];
#pragma unroll
    for (int k = 0; k < 5; k++) {
        inc[k] = x[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc[k], o);
            if (lane >= o) inc[k] += y;
        }
        if (lane == 31) ws[warp][k] = inc[k];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
        for (int k = 0; k < 5; k++) {
            int y = ws[lane][k];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int z = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) y += z;
            }
            ws[lane][k] = y;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 5; k++) {
        tot[k] = ws[31][k];
        x[k] = (warp ? ws[warp - 1][k] : 0) + inc[k] - x[k];
    }
}

__device__ __forceinline__ int tiles_of(int n_new, int group) {
    return (n_new * group + PG_TILE_ROWS - 1) / PG_TILE_ROWS;
}

// The last r with prefix[r] <= i, of an exclusive sum prefix[0..n] with prefix[n] > i.
__device__ __forceinline__ int owner(const int32_t* prefix, int n, int i) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// Everything but the per-request sums: one thread per token, unit and item, each finding its
// request by bisection of the exclusive sums (which skips requests that have none).
__device__ void plan_fill(const PlanArgs& a, int64_t tid, int64_t threads) {
    const jv_paged_batch& b = a.b;
    const int R = b.requests;
    const int32_t *unit_pre = a.v.prefix + (R + 1), *small_pre = unit_pre + (R + 1), *large_pre = small_pre + (R + 1);
    const int tokens = b.starts[R];
    for (int64_t t = tid; t < tokens; t += threads) {
        const int r = owner(b.starts, R, (int)t);
        const int n_new = b.starts[r + 1] - b.starts[r];
        const int pos = b.lengths[r] - n_new + (int)t - b.starts[r];
        b.request_of[t] = r;
        b.positions[t] = pos;
        b.slots[t] = (int64_t)b.block_table[(int64_t)r * b.max_blocks + pos / PG_TOKENS] * PG_TOKENS + pos % PG_TOKENS;
    }
    for (int64_t i = tid; i < unit_pre[R]; i += threads) {
        const int r = owner(unit_pre, R, (int)i);
        const int old = b.lengths[r] - (b.starts[r + 1] - b.starts[r]);
        a.v.units[i] = make_int2(r, old / PG_BLOCK + (int)i - unit_pre[r]);
    }
    for (int64_t i = tid; i < small_pre[R]; i += threads) {
        const int r = owner(small_pre, R, (int)i);
        a.v.small_items[i] = make_int4(r, (int)i - small_pre[r], small_pre[r + 1] - small_pre[r], 0);
    }
    for (int64_t i = tid; i < large_pre[R]; i += threads) {
        const int r = owner(large_pre, R, (int)i);
        // a request's last tile sees the most keys: first
        a.v.large_items[i] = make_int4(r, large_pre[r + 1] - 1 - (int)i, 0, 0);
    }
}

// One CTA: the sums over the requests, the checks, the new pages. Latency-bound: each thread holds
// up to 4 consecutive requests, one block-wide scan of five counts.
__global__ void __launch_bounds__(PLAN_THREADS) k_plan(PlanArgs a, bool fill) {
    __shared__ int ws[32][5];
    __shared__ unsigned long long keys_total, token_total;
    __shared__ int bad_code, bad_site;
    const jv_paged_batch& b = a.b;
    const int R = b.requests, tid = threadIdx.x;
    if (tid == 0) {
        keys_total = token_total = 0;
        bad_code = bad_site = 0;
    }
    __syncthreads();
    const int per = (R + PLAN_THREADS - 1) / PLAN_THREADS;  // <= 4
    const int r0 = tid * per;
    int old[4], n_new[4], cnt[4][5], sum[5] = {0, 0, 0, 0, 0};
    long long keys = 0, tokens = 0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        old[j] = n_new[j] = 0;
        if (j < per && r0 + j < R) {
            old[j] = a.cached[r0 + j];
            n_new[j] = a.new_tokens[r0 + j];
        }
        if (old[j] < 0 || n_new[j] < 0 || n_new[j] > b.max_new ||
            (long long)old[j] + n_new[j] > (long long)b.max_blocks * PG_TOKENS)
            bad = true;
        keys += (long long)old[j] + n_new[j];
        tokens += n_new[j];
    }
    if (bad) {
        if (atomicCAS(&bad_code, 0, JV_ERR_RANGE) == 0) bad_site = PS_PLAN_LENGTH;
        keys = tokens = 0;
    }
    atomicAdd(&keys_total, (unsigned long long)keys);
    atomicAdd(&token_total, (unsigned long long)tokens);
    __syncthreads();
    if (tid == 0 && bad_code == 0) {
        if (token_total > (unsigned long long)b.max_tokens) {
            bad_code = JV_ERR_RANGE;
            bad_site = PS_PLAN_TOKENS;
        } else if (keys_total > (unsigned long long)b.max_keys) {
            bad_code = JV_ERR_RANGE;
            bad_site = PS_PLAN_KEYS;
        }
    }
    __syncthreads();
    const bool within = bad_code == 0;  // from here on every count fits its list
    const int n_free = *a.n_free;
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
        for (int k = 0; k < 5; k++) cnt[j][k] = 0;
        const int total = old[j] + n_new[j];
        if (!within || j >= per || r0 + j >= R) continue;
        cnt[j][0] = n_new[j];
        cnt[j][1] = (total + PG_TOKENS - 1) / PG_TOKENS - (old[j] + PG_TOKENS - 1) / PG_TOKENS;
        if (n_new[j] > 0) {
            cnt[j][2] = (total + PG_BLOCK - 1) / PG_BLOCK - old[j] / PG_BLOCK;
            if ((int64_t)n_new[j] * b.group <= PG_SMALL_ROWS)
                cnt[j][3] = pg_chunks(total);
            else
                cnt[j][4] = tiles_of(n_new[j], b.group);
        }
#pragma unroll
        for (int k = 0; k < 5; k++) sum[k] += cnt[j][k];
    }
    int tot[5], pre[5];
#pragma unroll
    for (int k = 0; k < 5; k++) pre[k] = sum[k];
    block_scan5(pre, tot, ws);
    if (tid == 0 && within && (n_free < 0 || tot[1] > n_free)) {
        bad_code = JV_ERR_OOM;
        bad_site = PS_PLAN_FREE;
    }
    __syncthreads();
    if (bad_code == 0)
        for (int i = tid; i < tot[1]; i += PLAN_THREADS)
            if ((unsigned)a.free_pages[n_free - 1 - i] >= (unsigned)b.pages) {
                atomicExch(&bad_site, PS_PLAN_PAGE);
                atomicExch(&bad_code, JV_ERR_RANGE);
            }
    __syncthreads();
    const bool ok = bad_code == 0;
    int32_t *page_pre = a.v.prefix, *unit_pre = page_pre + (R + 1), *small_pre = unit_pre + (R + 1),
            *large_pre = small_pre + (R + 1);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = r0 + j;
        if (j >= per || r >= R) continue;
        b.lengths[r] = ok ? old[j] + n_new[j] : old[j];
        b.starts[r] = ok ? pre[0] : 0;
        page_pre[r] = ok ? pre[1] : 0;
        unit_pre[r] = ok ? pre[2] : 0;
        small_pre[r] = ok ? pre[3] : 0;
        large_pre[r] = ok ? pre[4] : 0;
        a.v.first[r] = ok ? pre[3] : 0;
        if (ok) {
            const int have = (old[j] + PG_TOKENS - 1) / PG_TOKENS;
            // a request that takes many pages is served by the whole block below
            if (cnt[j][1] <= 4)
                for (int k = 0; k < cnt[j][1]; k++)
                    b.block_table[(int64_t)r * b.max_blocks + have + k] = a.free_pages[n_free - 1 - (pre[1] + k)];
        }
#pragma unroll
        for (int k = 0; k < 5; k++) pre[k] += cnt[j][k];
    }
    if (tid == 0) {
        b.starts[R] = ok ? tot[0] : 0;
        page_pre[R] = ok ? tot[1] : 0;
        unit_pre[R] = ok ? tot[2] : 0;
        small_pre[R] = ok ? tot[3] : 0;
        large_pre[R] = ok ? tot[4] : 0;
        a.v.head[0] = ok ? tot[3] : 0;
        a.v.head[1] = ok ? tot[4] : 0;
        a.v.head[2] = ok ? tot[2] : 0;
        *a.n_free_out = ok ? n_free - tot[1] : n_free;
        if (!ok) paged_report(b.status, bad_code, bad_site);
    }
    __syncthreads();
    if (ok)
        for (int i = tid; i < tot[1]; i += PLAN_THREADS) {
            const int r = owner(page_pre, R, i);
            if (page_pre[r + 1] - page_pre[r] <= 4) continue;  // written above
            const int old_len = b.lengths[r] - (b.starts[r + 1] - b.starts[r]);
            b.block_table[(int64_t)r * b.max_blocks + (old_len + PG_TOKENS - 1) / PG_TOKENS + i - page_pre[r]] =
                a.free_pages[n_free - 1 - i];
        }
    if (fill) {
        __syncthreads();
        plan_fill(a, tid, PLAN_THREADS);
    }
}

__global__ void __launch_bounds__(256) k_plan_fill(PlanArgs a) {
    plan_fill(a, (int64_t)blockIdx.x * blockDim.x + threadIdx.x, (int64_t)gridDim.x * blockDim.x);
}

// ------------------------------------------------------------ read-back

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight lanes per (slot, KV head, K or V) row of 128 values: 16 bytes in, 16 values out per lane.
// Bound by the bytes out (2 or 4 times the bytes in).
template <class T>
__global__ void __launch_bounds__(256) k_kv8_read(jv_kv8_cache c, const int64_t* __restrict__ slots, int n, T* __restrict__ k_out,
                                                  T* __restrict__ v_out, int64_t row_stride, bool vec, int32_t* status) {
    const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const int part = threadIdx.x & 7;
    const int per = 2 * c.kv_heads;
    const int64_t at = i / per;
    if (at >= n) return;
    const int h = (int)(i % per) >> 1, kv = (int)(i % per) & 1;
    const int64_t slot = slots[at];
    if (slot < 0) return;
    const int64_t page = slot / PG_TOKENS;
    const int row = (int)(slot % PG_TOKENS);
    if (page >= c.pages) {
        paged_report(status, JV_ERR_RANGE, PS_READ_SLOT);
        return;
    }
    const int4 raw = *(const int4*)((const char*)c.data + page * c.page_bytes + (int64_t)(h * 2 + kv) * PG_PLANE + row * PG_DIM +
                                    part * 16);
    const float s = c.scales[page * c.scale_stride + (h * 2 + kv) * 4 + row / PG_BLOCK];
    T* dst = (kv ? v_out : k_out) + at * row_stride + h * PG_DIM + part * 16;
    alignas(16) T out[16];
    bool bad = false;
    const int w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const float x = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * s;
        if (sizeof(T) == 2 && std::is_same<T, __half>::value) bad |= f16_out_of_range(x);
        out[e] = from_f32<T>(x);
    }
    if (vec) {
#pragma unroll
        for (int e = 0; e < (int)sizeof(T); e++) ((uint4*)dst)[e] = ((const uint4*)out)[e];
    } else {
#pragma unroll
        for (int e = 0; e < 16; e++) dst[e] = out[e];
    }
    if (bad) paged_report(status, JV_ERR_NUMERIC, PS_READ_VALUE);
}

template <class T>
void launch_read(const jv_kv8_cache& c, const int64_t* slots, int n, void* k, void* v, int64_t stride, int32_t* status,
                 cudaStream_t s) {
    const bool vec = aligned(k, 16) && aligned(v, 16) && stride * sizeof(T) % 16 == 0;
    const int64_t threads = (int64_t)n * 2 * c.kv_heads * 8;
    k_kv8_read<T><<<(unsigned)((threads + 255) / 256), 256, 0, s>>>(c, slots, n, (T*)k, (T*)v, stride, vec, status);
    JV_CUDA(cudaGetLastError());
    note_launch();
}

}  // namespace
}  // namespace jv

using namespace jv;

extern "C" {

int64_t jv_paged_work_bytes(const jv_paged_batch* batch) {
    int64_t n = -1;
    paged_api([&] {
        check_batch(batch, false);
        n = plan_view(*batch).bytes;
    });
    return n;
}

int jv_paged_plan(const jv_paged_batch* batch, const int32_t* cached, const int32_t* new_tokens, const int32_t* free_pages,
                  const int32_t* n_free, int32_t* n_free_out, void* stream) {
    return paged_api([&] {
        check_batch(batch, true);
        if (!cached || !new_tokens || !free_pages || !n_free || !n_free_out) throw Error(JV_ERR_ARG, "NULL buffer");
        OnDeviceOf dev(batch->work);
        PlanArgs a{*batch, plan_view(*batch), cached, new_tokens, free_pages, n_free, n_free_out};
        // One CTA fills the arrays too where they are short enough that a second launch would cost
        // more than its parallelism saves.
        const int64_t rows = a.v.unit_cap + a.v.small_cap + a.v.large_cap + batch->max_tokens;
        const bool fill = rows <= 4096;
        k_plan<<<1, PLAN_THREADS, 0, (cudaStream_t)stream>>>(a, fill);
        JV_CUDA(cudaGetLastError());
        note_launch();
        if (!fill) {
            const int64_t ctas = std::min<int64_t>((batch->max_tokens + 255) / 256, 4 * 148);
            k_plan_fill<<<(unsigned)ctas, 256, 0, (cudaStream_t)stream>>>(a);
            JV_CUDA(cudaGetLastError());
            note_launch();
        }
    });
}

int jv_kv8_read(const jv_kv8_cache* cache, const int64_t* slots, int32_t n, int32_t type, void* k_out, void* v_out,
                int64_t row_stride, int32_t* status, void* stream) {
    return paged_api([&] {
        check_cache(cache);
        if (type_bytes(type) == 0) throw Error(JV_ERR_UNSUPPORTED, "the type must be F32 (0), F16 (1) or BF16 (30)");
        if (n < 0) throw Error(JV_ERR_ARG, "n is negative");
        if (n == 0) return;
        if (!slots || !k_out || !v_out) throw Error(JV_ERR_ARG, "NULL buffer");
        if (row_stride < (int64_t)cache->kv_heads * PG_DIM) throw Error(JV_ERR_ARG, "row_stride must be at least kv_heads * 128");
        if (!aligned(slots, 8) || !aligned(k_out, type_bytes(type)) || !aligned(v_out, type_bytes(type)))
            throw Error(JV_ERR_ARG, "a buffer is not aligned to its elements");
        if ((int64_t)n * 2 * cache->kv_heads * 8 / 256 > INT32_MAX - 1) throw Error(JV_ERR_RANGE, "too many slots for one call");
        OnDeviceOf dev(cache->data);
        cudaStream_t s = (cudaStream_t)stream;
        if (type == T_F32)
            launch_read<float>(*cache, slots, n, k_out, v_out, row_stride, status, s);
        else if (type == T_F16)
            launch_read<__half>(*cache, slots, n, k_out, v_out, row_stride, status, s);
        else
            launch_read<__nv_bfloat16>(*cache, slots, n, k_out, v_out, row_stride, status, s);
    });
}

}  // extern "C"
