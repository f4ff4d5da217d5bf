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
    // a small item is two entries of its list, which the plan indexes in 32 bits
    need(plan_view(*b).small_cap < (1 << 30), "the batch's bounds allow 2^30 work items or more");
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
    need(c->page_bytes < ((int64_t)1 << 40), "page_bytes must be below 2^40");
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
    // small items: a chunk has at least 64 keys except a request's last, 128 where a request has over 32 chunks, and
    // a request has at most 512 chunks up to 2^19 keys (pg_chunk_keys); units: every one holds a
    // new token, and a request's span has at most new / 16 + 2 of them
    const int64_t tiles = (std::min<int64_t>(PG_SMALL_ROWS, (int64_t)b.max_new * b.group) + PG_ROW_TILE - 1) / PG_ROW_TILE;
    const int64_t most = (int64_t)b.max_blocks * PG_TOKENS;  // of one request's keys
    const int64_t per = most <= 4096 ? std::min<int64_t>(32, (most + PG_CHUNK - 1) / PG_CHUNK) : std::max<int64_t>(512, (most + 2047) / 2048);
    v.small_cap = std::min(R + std::min(b.max_keys / PG_CHUNK, 32 * R + b.max_keys / 128), R * per) * tiles;
    const int64_t large = (int64_t)b.max_new * b.group > PG_SMALL_ROWS ? std::min<int64_t>(R, T * b.group / (PG_SMALL_ROWS + 1)) : 0;
    // at most PG_SPLIT_ITEMS / pairs splits of each of up to a quarter as many pairs, and a split has at least 1024
    // keys but for a request's last
    v.split_cap = std::min(PG_SPLIT_ITEMS * large, PG_SPLIT_ITEMS / 4 * (large + b.max_keys / 1024));
    v.large_cap = large ? v.split_cap + large + T / pg_pair_tokens(b.group) : 0;
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
    v.prefix = (int32_t*)take(4 * R * 4);
    v.small_items = (int4*)take(v.small_cap * 32);
    v.large_items = (int4*)take(v.large_cap * 16);
    v.large_rows = (int4*)take(v.large_cap * 16);
    v.units = (int4*)take(v.unit_cap * 16);
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
constexpr int PLAN_PER = PG_MAX_REQUESTS / PLAN_THREADS;  // requests per thread at most
constexpr int PLAN_FILL_THREADS = 128;
constexpr int PLAN_FILL_REQUESTS = 256;  // most requests that the first launch fills for

// A request's place in the batch: its lengths and the exclusive sums in front of it.
struct Place {
    int old, n_new, start, page, unit, small, large, split;  // split: large items with more than one split
};

__device__ __forceinline__ int units_of(int old, int n_new) {
    return n_new > 0 ? (old + n_new + PG_BLOCK - 1) / PG_BLOCK - old / PG_BLOCK : 0;
}
__device__ __forceinline__ int pages_of(int old, int n_new) {
    return (old + n_new + PG_TOKENS - 1) / PG_TOKENS - (old + PG_TOKENS - 1) / PG_TOKENS;
}
__device__ __forceinline__ bool is_small(int n_new, int group) { return (int64_t)n_new * group <= PG_SMALL_ROWS; }
__device__ __forceinline__ int small_of(int old, int n_new, int group) {
    return n_new > 0 && is_small(n_new, group) ? pg_chunks(old + n_new, n_new * group) * ((n_new * group + PG_ROW_TILE - 1) / PG_ROW_TILE) : 0;
}
__device__ __forceinline__ int large_of(int old, int n_new, int group) {
    return n_new > 0 && !is_small(n_new, group) ? pg_pairs(n_new, group) * pg_splits(old + n_new, pg_pairs(n_new, group)) : 0;
}

// One request's pages, tokens, units and items, by threads t, t + n, ...
__device__ __forceinline__ void plan_request(const PlanArgs& a, int r, const Place& q, int n_free, int t, int n) {
    const jv_paged_batch& b = a.b;
    int32_t* row = b.block_table + (int64_t)r * b.max_blocks;
    const int have = (q.old + PG_TOKENS - 1) / PG_TOKENS, pages = pages_of(q.old, q.n_new);
    for (int k = t; k < pages; k += n) row[have + k] = a.free_pages[n_free - 1 - (q.page + k)];
    for (int i = t; i < q.n_new; i += n) {
        const int pos = q.old + i, blk = pos / PG_TOKENS;
        // a page of this step comes from where it is taken, so that no thread waits for another's write
        const int page = blk >= have ? a.free_pages[n_free - 1 - (q.page + blk - have)] : row[blk];
        b.request_of[q.start + i] = r;
        b.positions[q.start + i] = pos;
        b.slots[q.start + i] = (int64_t)page * PG_TOKENS + pos % PG_TOKENS;
    }
    const int units = units_of(q.old, q.n_new);
    for (int i = t; i < units; i += n) {
        const int block = q.old / PG_BLOCK + i, p0 = block * PG_BLOCK;
        const int lo = max(0, q.old - p0), hi = min(PG_BLOCK, q.old + q.n_new - p0);
        a.v.units[q.unit + i] = make_int4(r, block, q.start + p0 - q.old, lo | hi << 8);
    }
    const int small = small_of(q.old, q.n_new, b.group), chunks = pg_chunks(q.old + q.n_new, q.n_new * b.group);
    for (int i = t; i < small; i += n) {
        a.v.small_items[2 * (q.small + i)] = make_int4(r, i % chunks, chunks, i / chunks);
        a.v.small_items[2 * (q.small + i) + 1] = make_int4(q.start, q.n_new, q.old + q.n_new, 0);
    }
    const int large = large_of(q.old, q.n_new, b.group), pairs = pg_pairs(q.n_new, b.group);
    const int splits = large > 0 ? large / pairs : 1;
    // a request's last tiles see the most keys: first
    for (int i = t; i < large; i += n) {
        a.v.large_items[q.large + i] = make_int4(r, pairs - 1 - i / splits, i % splits, splits | (splits > 1 ? (q.split + i) << 8 : 0));
        a.v.large_rows[q.large + i] = make_int4(q.start, q.n_new, q.old + q.n_new, 0);
    }
}

// One CTA: the sums over the requests and the checks; with `fill`, everything else too, a warp per
// request. Latency-bound: each thread holds up to 4 consecutive requests, the sums are one pass of
// warp shuffles and one barrier (every warp adds up the warps' totals for itself).
__global__ void __launch_bounds__(PLAN_THREADS) k_plan(PlanArgs a, bool fill) {
    __shared__ int ws[32][6];
    __shared__ long long wl[32][2];
    __shared__ Place places[PLAN_FILL_REQUESTS];
    pdl_wait();
    pdl_launch_dependents();
    const jv_paged_batch& b = a.b;
    const int R = b.requests, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int per = (R + blockDim.x - 1) / blockDim.x, r0 = tid * per;  // per <= PLAN_PER
    const int n_free = *a.n_free;
    int old[PLAN_PER], n_new[PLAN_PER], sum[6] = {0, 0, 0, 0, 0, 0};
    long long keys = 0, tokens = 0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < PLAN_PER; j++) {
        const bool in = j < per && r0 + j < R;
        old[j] = in ? a.cached[r0 + j] : 0;
        n_new[j] = in ? a.new_tokens[r0 + j] : 0;
    }
#pragma unroll
    for (int j = 0; j < PLAN_PER; j++) {
        if (j >= per) break;
        const long long total = (long long)old[j] + n_new[j];
        if (old[j] < 0 || n_new[j] < 0 || n_new[j] > b.max_new || total > (long long)b.max_blocks * PG_TOKENS) {
            bad = true;  // the step fails; its counts are left out
            continue;
        }
        keys += total;
        tokens += n_new[j];
        sum[0] += n_new[j];
        sum[1] += pages_of(old[j], n_new[j]);
        sum[2] += units_of(old[j], n_new[j]);
        sum[3] += small_of(old[j], n_new[j], b.group);
        const int large = large_of(old[j], n_new[j], b.group);
        sum[4] += large;
        sum[5] += large > pg_pairs(n_new[j], b.group) ? large : 0;
    }
    int pre[6];
#pragma unroll
    for (int k = 0; k < 6; k++) {
        int x = sum[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) ws[warp][k] = x;
        pre[k] = x - sum[k];
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        keys += __shfl_xor_sync(0xffffffffu, keys, o);
        tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
    }
    if (lane == 0) wl[warp][0] = keys, wl[warp][1] = tokens;
    bad = __syncthreads_or(bad);
    int tot[6];
    {
        int before[6];
#pragma unroll
        for (int k = 0; k < 6; k++) {
            const int x = lane < warps ? ws[lane][k] : 0;
            before[k] = lane < warp ? x : 0;
            tot[k] = x;
        }
        keys = lane < warps ? wl[lane][0] : 0;
        tokens = lane < warps ? wl[lane][1] : 0;
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) {
#pragma unroll
            for (int k = 0; k < 6; k++) {
                before[k] += __shfl_xor_sync(0xffffffffu, before[k], o);
                tot[k] += __shfl_xor_sync(0xffffffffu, tot[k], o);
            }
            keys += __shfl_xor_sync(0xffffffffu, keys, o);
            tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
        }
#pragma unroll
        for (int k = 0; k < 6; k++) pre[k] += before[k];
    }
    int code = 0, site = 0;  // the same in every thread
    if (bad)
        code = JV_ERR_RANGE, site = PS_PLAN_LENGTH;
    else if (tokens > b.max_tokens)
        code = JV_ERR_RANGE, site = PS_PLAN_TOKENS;
    else if (keys > b.max_keys)
        code = JV_ERR_RANGE, site = PS_PLAN_KEYS;
    else if (n_free < 0 || tot[1] > n_free)
        code = JV_ERR_OOM, site = PS_PLAN_FREE;
    if (code == 0) {
        bool out = false;
        for (int i = tid; i < tot[1]; i += blockDim.x) out |= (unsigned)a.free_pages[n_free - 1 - i] >= (unsigned)b.pages;
        if (__syncthreads_or(out)) code = JV_ERR_RANGE, site = PS_PLAN_PAGE;
    }
    const bool ok = code == 0;
    int32_t* prefix = a.v.prefix;
#pragma unroll
    for (int j = 0; j < PLAN_PER; j++) {
        const int r = r0 + j;
        if (j >= per) break;
        if (r >= R) continue;
        const Place q = {old[j], ok ? n_new[j] : 0, ok ? pre[0] : 0, ok ? pre[1] : 0, ok ? pre[2] : 0, ok ? pre[3] : 0, ok ? pre[4] : 0,
                         ok ? pre[5] : 0};
        b.lengths[r] = q.old + q.n_new;
        b.starts[r] = q.start;
        a.v.first[r] = q.small;
        if (fill) {
            places[r] = q;
        } else {
            prefix[r] = q.page;
            prefix[R + r] = q.unit;
            prefix[2 * R + r] = q.large;
            prefix[3 * R + r] = q.split;
        }
        pre[0] += n_new[j];
        pre[1] += pages_of(old[j], n_new[j]);
        pre[2] += units_of(old[j], n_new[j]);
        pre[3] += small_of(old[j], n_new[j], b.group);
        const int large = large_of(old[j], n_new[j], b.group);
        pre[4] += large;
        pre[5] += large > pg_pairs(n_new[j], b.group) ? large : 0;
    }
    if (tid == 0) {
        b.starts[R] = ok ? tot[0] : 0;
        a.v.head[0] = ok ? tot[3] : 0;
        a.v.head[1] = ok ? tot[4] : 0;
        a.v.head[2] = ok ? tot[2] : 0;
        a.v.head[3] = n_free;
        *a.n_free_out = ok ? n_free - tot[1] : n_free;
        if (!ok) paged_report(b.status, code, site);
    }
    if (fill && ok) {
        __syncthreads();
        for (int r = warp; r < R; r += warps)
            if (places[r].n_new > 0) plan_request(a, r, places[r], n_free, lane, 32);
    }
}

// The rest of a larger step: a CTA per request and slice of its tokens.
__global__ void __launch_bounds__(PLAN_FILL_THREADS) k_plan_fill(PlanArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    const jv_paged_batch& b = a.b;
    const int r = blockIdx.x, R = b.requests;
    const int len = b.lengths[r], start = b.starts[r], n_new = b.starts[r + 1] - start;
    const Place q = {len - n_new, n_new, start, a.v.prefix[r], a.v.prefix[R + r], a.v.first[r], a.v.prefix[2 * R + r],
                     a.v.prefix[3 * R + r]};
    const int n_free = a.v.head[3];
    if (n_new > 0) plan_request(a, r, q, n_free, blockIdx.y * PLAN_FILL_THREADS + threadIdx.x, gridDim.y * PLAN_FILL_THREADS);
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
    pdl_wait();
    pdl_launch_dependents();
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

// One CTA: a block and a slice of its planes, two planes at a time. Bound by HBM: up to 26 MB in and out for 64
// requests on 26 layers of 8 KV heads, which added 10 us at most to a pass of 6.56 ms.
constexpr int SAVE_THREADS = 256;
__global__ void __launch_bounds__(SAVE_THREADS) k_kv8_save_blocks(PagePlanes c, const int4* __restrict__ blocks, uint8_t* saved, bool restore) {
    pdl_wait();
    pdl_launch_dependents();
    const int4 b = blocks[blockIdx.x];
    if ((unsigned)b.x >= (unsigned)c.pages || b.y < 0 || b.z < 0 || b.z > PG_BLOCK || b.y > PG_TOKENS - PG_BLOCK) return;
    const int i = threadIdx.x & 127;  // 16 bytes of the block's rows
    for (int p = blockIdx.y * 2 + (threadIdx.x >> 7); p < c.planes; p += gridDim.y * 2) {
        uint8_t* at = c.data + b.x * c.page_bytes + (int64_t)p * PG_PLANE + b.y * PG_DIM;
        float* scale = c.scales + b.x * c.scale_stride + 4 * (int64_t)p + b.y / PG_BLOCK;
        uint8_t* kept = saved + ((int64_t)blockIdx.x * c.planes + p) * PG_SAVED;
        if (i * 16 < b.z * PG_DIM) {
            uint4* x = (uint4*)(at + i * 16);
            uint4* y = (uint4*)(kept + i * 16);
            restore ? *x = *y : *y = *x;
        }
        if (i == 0) {
            float* y = (float*)(kept + PG_BLOCK * PG_DIM);
            restore ? *scale = *y : *y = *scale;
        }
    }
}

template <class T>
void launch_read(const jv_kv8_cache& c, const int64_t* slots, int n, void* k, void* v, int64_t stride, int32_t* status,
                 cudaStream_t s) {
    const bool vec = aligned(k, 16) && aligned(v, 16) && stride * sizeof(T) % 16 == 0;
    const int64_t threads = (int64_t)n * 2 * c.kv_heads * 8;
    launch_pdl(k_kv8_read<T>, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, c, slots, n, (T*)k, (T*)v, stride, vec, status);
    note_launch();
}

}  // namespace

void launch_kv8_save_blocks(const PagePlanes& c, const int4* blocks, int n, uint8_t* saved, bool restore, cudaStream_t s) {
    launch_pdl(k_kv8_save_blocks, dim3(n, (c.planes + 7) / 8), dim3(SAVE_THREADS), 0, s, c, blocks, saved, restore);
    note_launch();
}

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
        // A CTA of few warps for few requests. It fills the arrays too where a warp per request gets
        // through them in less than a second launch costs (16 requests of one token: 6.8 us in one launch).
        const bool fill = batch->requests <= PLAN_FILL_REQUESTS && batch->max_new <= 256 && batch->max_tokens <= 4096;
        const int threads = batch->requests <= 8 ? 256 : PLAN_THREADS;
        launch_pdl(k_plan, dim3(1), dim3(threads), 0, (cudaStream_t)stream, a, fill);
        note_launch();
        if (!fill) {
            const int slices = std::min(32, (batch->max_new + 1023) / 1024);
            launch_pdl(k_plan_fill, dim3(batch->requests, slices), dim3(PLAN_FILL_THREADS), 0, (cudaStream_t)stream, a);
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
