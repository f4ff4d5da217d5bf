// paged.h — what the paged-batch operators (paged.cu, kernels_rope.cu, kv8_attn.cu) share: the
// layout of the 8-bit cache and of a plan's work lists, and the host-side checks.
#pragma once

#include <type_traits>

#include "jv_internal.h"

namespace jv {

constexpr int PG_TOKENS = JV_PAGE_TOKENS;          // tokens per page
constexpr int PG_BLOCK = JV_SCALE_TOKENS;          // tokens per scale
constexpr int PG_DIM = 128;                        // head_dim
constexpr int PG_PLANE = PG_TOKENS * PG_DIM;       // bytes of one K or V plane of a page
constexpr int PG_MAX_REQUESTS = 4096;
constexpr int PG_MAX_GROUP = 16;

// A request whose new tokens x group give at most PG_SMALL_ROWS query rows is "small": its keys are
// split into chunks that different warps take, PG_ROW_TILE rows at a time (kv8_attn.cu). The others go by
// pairs of 128-row tiles to the tensor cores (kv8_attn_tc.cu).
constexpr int PG_SMALL_ROWS = 32;
constexpr int PG_ROW_TILE = 16;
constexpr int PG_TILE = 128;  // query rows of a tensor-core tile; a large item is two tiles

// Keys per chunk of a small request: 64 up to 2048 keys, where latency counts; then as many as keep what a
// chunk leaves behind (rows x 528 bytes, written and read again) small against its keys, which with more than
// 8 rows begins earlier. It goes by the request's own length and rows, so a request is cut alike in every
// batch. Always a multiple of 64, at most 2048 (32 pages: one per lane).
constexpr int PG_CHUNK = 64;
__host__ __device__ inline int pg_chunk_keys(int len, int rows) {
    if (len <= (rows > 8 ? 512 : 2048)) return PG_CHUNK;
    if (len <= (rows > 8 ? 1024 : 4096)) return 128;
    return len <= 131072 ? 256 : len <= 524288 ? 1024 : 2048;
}
__host__ __device__ inline int pg_chunks(int len, int rows) {
    return len <= 0 ? 0 : (int)(((int64_t)len + pg_chunk_keys(len, rows) - 1) / pg_chunk_keys(len, rows));
}

// The scale that a block of zero values (scale 0) counts as in attention. Its values are 0 at any scale, so only the
// softmax's denominator takes it, in fp32; but log2 of it enters the exponents of which the largest is a row's
// reference M, and a stand-in above the scales around it would push their fp16 weights down into subnormals (at 1,
// values of 1e-4 beside zeros were 3 % off, and gone where the zeros' keys scored 2^8 above theirs). So it is below any
// scale that values of 2^-50 or more come with, and beside values up to 2^40 weights down to 2^-32 of the largest are still an fp32.
constexpr float PG_ZERO_SCALE = 0x1p-60f;

// Tokens of a large item (two tiles of 128 / group tokens), and the items of a request: its keys are split
// too, in parts of at least 1024 keys, where it has at most 4 pairs of tiles: up to 16 items. By the request's own
// sizes again. The parts go by the whole length, also in a window, where most of them then have no block: the end at
// 4 pairs was measured there (five chunks of 100 to 1500 tokens in a window of 4096: 285 us, 317 with up to 16 items
// for up to 8 pairs, 461 with 32). For a lone request without a window it is a cliff: 256 tokens on 30,000 keys
// take 173 us, 257 tokens 543.
constexpr int PG_SPLIT_ITEMS = 16;  // a split of a pair is joined by a lane each
__host__ __device__ inline int pg_pair_tokens(int group) { return 2 * (PG_TILE / group); }
__host__ __device__ inline int pg_pairs(int n_new, int group) { return (n_new + pg_pair_tokens(group) - 1) / pg_pair_tokens(group); }
__host__ __device__ inline int pg_splits(int len, int pairs) {
    if (pairs > PG_SPLIT_ITEMS / 4) return 1;
    const int blocks = (int)(((int64_t)len + 127) / 128), most = (blocks + 7) / 8;
    return most < 1 ? 1 : most < PG_SPLIT_ITEMS / pairs ? most : PG_SPLIT_ITEMS / pairs;
}

// A plan's work lists, in jv_paged_batch.work.
struct PlanView {
    int32_t* head;      // [8]: small items, large items, append units, free pages before the step
    int32_t* first;     // [requests] first small item of each request
    int32_t* prefix;    // [4][requests]: pages taken, units, large items and those with splits before request r
    int4* small_items;  // two each: {request, chunk, chunks, row tile}, {start, new, length, 0}; row tile by row tile
    int4* large_items;  // {request, pair of tiles, split, splits + 256 x place of its partials}; a pair's splits next to each other
    int4* large_rows;   // beside each: {start, new, length, 0} of its request
    int4* units;        // the 16-token blocks the step writes to: {request, block, token of its row 0, first new row + 256 x end}
    int64_t small_cap, large_cap, split_cap, unit_cap, bytes;  // split_cap: most large items with more than one split
};
PlanView plan_view(const jv_paged_batch& b);

// A page's planes of all layers, heads, K and V: plane p is int8 [64][128] at data + page * page_bytes + p * PG_PLANE,
// its scales fp32 [4] at scales + page * scale_stride + 4 p.
struct PagePlanes {
    uint8_t* data;
    float* scales;
    int64_t page_bytes, scale_stride;
    int pages, planes;
};
// Rows [y, y + z) of page x, less than a block of 16: the tokens of a request in the block that its next token
// continues. An append to the block may round them again, so who must be able to take a step back copies them (and
// the block's scale) to `saved`, n * planes * PG_SAVED bytes, and from there.
constexpr int PG_SAVED = PG_BLOCK * PG_DIM + 16;
void launch_kv8_save_blocks(const PagePlanes& c, const int4* blocks, int n, uint8_t* saved, bool restore, cudaStream_t s);

void check_batch(const jv_paged_batch* b, bool arrays);
void check_cache(const jv_kv8_cache* c);
void check_rows(const jv_heads* x, const char* name, int dim, int64_t tokens);
int type_bytes(int type);  // 0 for a type the operators do not take

// Runs on the device that `p` is on, for the guard's lifetime.
struct OnDeviceOf {
    int before = -1;
    explicit OnDeviceOf(const void* p);
    ~OnDeviceOf();
    OnDeviceOf(const OnDeviceOf&) = delete;
};

template <class F>
int paged_api(F&& f) {
    try {
        f();
        return JV_OK;
    } catch (const Error& e) {
        return api_error(e.code, e.what());
    } catch (const std::exception& e) {
        return api_error(JV_ERR_ARG, e.what());
    } catch (...) {
        return api_error(JV_ERR_ARG, "an unknown error");
    }
}

// Sites of the status word (word 1).
enum PagedSite : int {
    PS_PLAN_LENGTH = 96, PS_PLAN_TOKENS = 97, PS_PLAN_KEYS = 98, PS_PLAN_FREE = 99, PS_PLAN_PAGE = 100,
    PS_APPEND_PAGE = 101, PS_APPEND_VALUE = 102, PS_READ_SLOT = 103, PS_READ_VALUE = 104,
    PS_ATTN_VALUE = 105, PS_ATTN_PAGE = 106, PS_ROPE_VALUE = 107, PS_ATTN_WAIT = 108, PS_ATTN_TC = 112 /* + role */
};

// An attention launch.
struct AttnKArgs {
    jv_kv8_cache c;
    jv_paged_batch b;
    PlanView v;
    jv_heads q;
    float scale;  // times log2 e
    int window;
    float* part_o;    // [small item][kv head][rows][128]
    float2* part_ml;  // [small item][kv head][rows]
    int rows;         // query rows of a small item's partials
    float* large_o;   // [large item with splits][kv head][256][128]
    float2* large_ml; // [large item with splits][kv head][256]
};
// Large requests, and the joining of their splits (kv8_attn_tc.cu).
void launch_kv8_large(const AttnKArgs& a, int type, cudaStream_t s);

#ifdef __CUDACC__
__device__ __forceinline__ void paged_report(int32_t* status, int code, int site) {
    if (!status) return;
    if (atomicCAS(status, 0, code) == 0) atomicExch(status + 1, site);
}

// Outputs about to be rounded to T: whether one becomes an fp16 infinity or is not a number.
template <class T>
__device__ __forceinline__ bool outside(float4 o) {
    return std::is_same<T, __half>::value &&
           (f16_out_of_range(o.x) || f16_out_of_range(o.y) || f16_out_of_range(o.z) || f16_out_of_range(o.w));
}

// The request's rows of a plan, as an operator after it uses them; false (and a report) where the
// arrays do not hold what a plan writes.
struct RequestRows {
    int start, n_new, len;
};
__device__ __forceinline__ bool rows_in_bounds(const jv_paged_batch& b, int start, int n_new, int len) {
    return start >= 0 && n_new >= 0 && n_new <= b.max_new && start <= b.max_tokens - n_new && len >= 0 &&
           len <= (int64_t)b.max_blocks * PG_TOKENS;
}
__device__ __forceinline__ bool request_rows(const jv_paged_batch& b, int r, RequestRows& o) {
    if (r < 0 || r >= b.requests) return false;
    o.start = b.starts[r];
    o.n_new = b.starts[r + 1] - o.start;
    o.len = b.lengths[r];
    return rows_in_bounds(b, o.start, o.n_new, o.len);
}
#endif

}  // namespace jv
