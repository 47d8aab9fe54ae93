// kt_paged.cu -- the paged 16-bit key/value cache: new tokens, rotated by their
// positions, into their pages; the accepted path of a drafted tree; the C entries.
#include <algorithm>
#include <cmath>

#include "kt_paged.h"

namespace kt {
namespace {

constexpr int kThreads = 128;
constexpr int kMostNodes = 1024;  // of a drafted tree
constexpr int kMostPairs = 64;    // of a head

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// ------------------------------------------------------------ append
//
// Row (b, t) at position p turns the pair (x, y) = (head[i], head[i + d/2]) of every query
// and key head by the angle p * inv_freq[i]:
//   x' = x cos - y sin,   y' = x sin + y cos.
// The angle's product is taken in 64 bits and brought into [-pi, pi] there: rounded to
// fp32, as the reference does, the product at position 100,000 would be off by up to 4e-3,
// twice what bf16 keeps.  A CTA has a row, whose sines it forms once; a thread four pairs of
// it, for which it goes over heads.  (A thread forming its own four for every head: 28.7 us
// where this takes 26.0, and a token of 64 sequences 3.1 where this takes 2.5.)
// Bound by memory for prompts: 4 x 1021 rows of 32 + 8 + 8 heads of 128 26.0 us, 5.8 TB/s; by
// latency for steps.

struct Append {
    const float *q, *k, *v, *inv_freq;
    const int32_t *counts, *depths;
    void* q_out;
    int32_t* status;
    int64_t q_stride, k_stride, v_stride;
    int32_t heads, rows, layer, aligned, each;  // each: heads a thread goes over
};

__device__ __forceinline__ void load4(const float* p, bool aligned, float (&x)[4]) {
    if (aligned) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = p[i];
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(Paged c, Append a) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int d = c.head_dim, half = d / 2, quads = half / 4;
    const int64_t r = blockIdx.x;
    const int b = static_cast<int>(blockIdx.x / static_cast<uint32_t>(a.rows)), t = static_cast<int>(blockIdx.x) - b * a.rows;
    const int at_once = kThreads / quads, quad = threadIdx.x % quads, first = threadIdx.x / quads;
    const int all = a.heads + 2 * c.kv_heads;
    const int begin = blockIdx.y * at_once * a.each + first, end = min(all, (static_cast<int>(blockIdx.y) + 1) * at_once * a.each);
    T* const q_out = static_cast<T*>(a.q_out) + r * a.heads * d + 4 * quad;
    const bool token = t < paged::rows_of(a.counts, b, a.rows);
    const int held = max(c.lengths[b], 0), shift = __ffs(c.page) - 1;
    const bool fits = static_cast<int64_t>(held) + t < static_cast<int64_t>(c.width) << shift;
    if (!token || !fits) {  // (past the last slot: dropped, and no token either)
        if (token && a.status != nullptr && threadIdx.x == 0 && blockIdx.y == 0) *a.status = KT_ERR_INVALID_ARGUMENT;
        if (first >= at_once) return;
        for (int h = begin; h < min(end, a.heads); h += at_once) {
            *reinterpret_cast<uint2*>(q_out + static_cast<int64_t>(h) * d) = make_uint2(0u, 0u);
            *reinterpret_cast<uint2*>(q_out + static_cast<int64_t>(h) * d + half) = make_uint2(0u, 0u);
        }
        return;
    }
    __shared__ float2 turn[kMostPairs];  // cosines and sines of the row's angles
    const int slot = held + t;
    const int page = c.table[static_cast<int64_t>(b) * c.table_stride + (slot >> shift)];
    const bool stored = page >= 0 && page < c.pages;
    if (!stored && a.status != nullptr && threadIdx.x == 0 && blockIdx.y == 0) *a.status = KT_ERR_INVALID_ARGUMENT;
    if (begin - first < a.heads + c.kv_heads) {  // as for the whole CTA
        if (threadIdx.x < half) {
            const double p = static_cast<double>(held) + static_cast<double>(a.depths ? a.depths[r] : t);
            const double angle = p * static_cast<double>(a.inv_freq[threadIdx.x]);
            const double turns = rint(angle * 0.15915494309189535);
            float sn, cs;
            sincosf(static_cast<float>(fma(-turns, 6.283185307179586, angle)), &sn, &cs);
            turn[threadIdx.x] = make_float2(cs, sn);
        }
        __syncthreads();
    }
    if (first >= at_once) return;
    float sn[4] = {}, cs[4] = {};
    if (begin < a.heads + c.kv_heads) {
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = turn[4 * quad + i].x, sn[i] = turn[4 * quad + i].y;
    }
    const int64_t layer = static_cast<int64_t>(a.layer) * c.pages;
    const int64_t row = ((layer + page) * c.kv_heads << shift) + (slot & (c.page - 1));  // of head 0
    // two heads at a time, so that the loads of one do not wait for the other's
    for (int h0 = begin; h0 < end; h0 += 2 * at_once) {
        float u[2][4], w[2][4];
        T* to[2] = {nullptr, nullptr};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int h = h0 + i * at_once;
            if (h >= end) continue;
            const float* from;
            if (h < a.heads) {
                from = a.q + r * a.q_stride + static_cast<int64_t>(h) * d;
                to[i] = q_out + static_cast<int64_t>(h) * d;
            } else {
                const bool key = h < a.heads + c.kv_heads;
                const int g = h - a.heads - (key ? 0 : c.kv_heads);
                from = (key ? a.k + r * a.k_stride : a.v + r * a.v_stride) + static_cast<int64_t>(g) * d;
                if (stored) to[i] = static_cast<T*>(key ? c.keys : c.values) + (row + static_cast<int64_t>(g) * c.page) * d + 4 * quad;
            }
            const bool aligned = a.aligned & (h < a.heads ? 1 : h < a.heads + c.kv_heads ? 2 : 4);
            load4(from + 4 * quad, aligned, u[i]);
            load4(from + 4 * quad + half, aligned, w[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (to[i] == nullptr) continue;
            if (h0 + i * at_once < a.heads + c.kv_heads) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = u[i][j], y = w[i][j];
                    u[i][j] = x * cs[j] - y * sn[j];
                    w[i][j] = x * sn[j] + y * cs[j];
                }
            }
            using H = paged::Half16<T>;
            *reinterpret_cast<uint2*>(to[i]) = make_uint2(H::pack(u[i][0], u[i][1]), H::pack(u[i][2], u[i][3]));
            *reinterpret_cast<uint2*>(to[i] + half) = make_uint2(H::pack(w[i][0], w[i][1]), H::pack(w[i][2], w[i][3]));
        }
    }
}

// ------------------------------------------------------------ accept
//
// Each CTA walks its sequence's tree again (a few dozen nodes in shared memory) and moves
// its layer's keys or values.  Node p_i of the path moves from slot n + p_i to n + i; p_i >= i
// and grows, so no move overwrites what a later one reads.
// Bound by latency: the tree, the places of the path's pages, the move, one after the other.

struct Accept {
    const int32_t *tokens, *parents, *choices, *counts;
    int32_t *accepted, *taken, *status;
    int32_t rows;
};

__global__ void __launch_bounds__(kThreads) paged_accept_kernel(Paged c, Accept a) {
    __shared__ int32_t token[kMostNodes], parent[kMostNodes], choice[kMostNodes], path[kMostNodes];
    __shared__ int nodes;
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const int b = blockIdx.y, rows = paged::rows_of(a.counts, b, a.rows);
    const int64_t line = static_cast<int64_t>(b) * a.rows;
    for (int i = threadIdx.x; i < rows; i += kThreads) {
        token[i] = a.tokens[line + i];
        parent[i] = a.parents[line + i];
        choice[i] = a.choices[line + i];
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int n = 0;
        for (int at = rows > 0 ? 0 : -1; at >= 0;) {
            if (lane == 0) path[n] = at;
            ++n;
            const int want = choice[at];
            int found = -1;
            for (int i = at + 1; i < rows && found < 0; i += 32) {  // children come after their parents
                const bool fits = i + lane < rows && parent[i + lane] == at && token[i + lane] == want;
                const uint32_t who = __ballot_sync(0xffffffffu, fits);
                if (who != 0) found = i + __ffs(who) - 1;
            }
            at = found;
        }
        if (lane == 0) nodes = n;
    }
    __syncthreads();
    const int n = nodes;
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < a.rows; i += kThreads) a.accepted[line + i] = i < n ? choice[path[i]] : -1;
        if (threadIdx.x == 0) a.taken[b] = n;
    }
    const int64_t held = max(c.lengths[b], 0);
    const int pieces = c.kv_heads * (c.head_dim / 8), per_head = c.head_dim / 8;
    uint4* const pool = static_cast<uint4*>(blockIdx.x % 2 ? c.values : c.keys) +
                        static_cast<int64_t>(blockIdx.x / 2) * c.pages * pieces * c.page;
    const int32_t* const table = c.table + static_cast<int64_t>(b) * c.table_stride;
    auto place = [&](int node) -> int64_t {  // of head 0, in pieces of 16 bytes; -1: no page
        const int64_t slot = held + node;
        if (slot >= static_cast<int64_t>(c.width) * c.page) return -1;
        const int page = table[slot / c.page];
        if (page < 0 || page >= c.pages) return -1;
        return (static_cast<int64_t>(page) * c.kv_heads * c.page + slot % c.page) * per_head;
    };
    constexpr int kBatch = 8;  // nodes whose places are looked up, and whose pieces are under way, together
    __shared__ int64_t from[kBatch], to[kBatch];
    for (int first = 0; first < n; first += kBatch) {
        const int many = min(kBatch, n - first);
        if (threadIdx.x < many) {
            const int i = first + threadIdx.x;
            const int64_t source = place(path[i]), target = place(i);
            const bool both = source >= 0 && target >= 0;
            if (!both && a.status != nullptr) *a.status = KT_ERR_INVALID_ARGUMENT;
            from[threadIdx.x] = both && path[i] != i ? source : -1;
            to[threadIdx.x] = target;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < pieces; e += kThreads) {
            const int64_t off = static_cast<int64_t>(e / per_head) * c.page * per_head + e % per_head;
            uint4 w[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (i < many && from[i] >= 0) w[i] = pool[from[i] + off];
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (i < many && from[i] >= 0) pool[to[i] + off] = w[i];
        }
        __syncthreads();
    }
}

const char* check(const Paged* c) {
    if (c == nullptr || !c->keys || !c->values || !c->table || !c->lengths) return "NULL argument";
    if (c->layers < 1 || c->pages < 1 || c->width < 1) return "layers, pages and width must be positive";
    if (c->batch < 1 || c->batch > 32767) return "batch must be in 1..32767";
    if (c->kv_heads < 1 || c->kv_heads > 65535) return "kv_heads must be in 1..65535";
    if (c->head_dim < 64 || c->head_dim > 128 || c->head_dim % 16 != 0) return "head_dim must be a multiple of 16 in 64..128";
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return "page must be 16, 32, 64 or 128";
    if (c->dtype != KT_BF16 && c->dtype != KT_FP16) return "dtype must be KT_BF16 or KT_FP16";
    if (c->table_stride < c->width) return "rows of the table are shorter than width";
    if (static_cast<int64_t>(c->width) * c->page > (1 << 30)) return "a sequence's pages hold at most 2^30 slots";
    if (static_cast<int64_t>(c->pages) * c->kv_heads * c->page > (1ll << 31) - 1) return "too many rows in a layer's pool";
    if (!aligned16(c->keys) || !aligned16(c->values)) return "keys and values must be 16-byte aligned";
    return nullptr;
}

// Whether the output (of `bytes`) shares memory with an input: `rows` of row_bytes, `stride`
// bytes apart.
bool overlaps(const void* out, int64_t bytes, const void* in, int64_t row_bytes, int64_t rows = 1, int64_t stride = 1) {
    if (out == nullptr || in == nullptr || bytes <= 0 || row_bytes <= 0 || rows <= 0) return false;
    const uintptr_t o = reinterpret_cast<uintptr_t>(out), i = reinterpret_cast<uintptr_t>(in), end = i + row_bytes;
    const int64_t first = o < end ? 0 : static_cast<int64_t>((o - end) / stride) + 1;  // the first row that ends behind o
    return first < rows && i + first * stride < o + bytes;
}
// The same for what every call reads of the cache's table and lengths.
bool overlaps_places(const void* out, int64_t bytes, const Paged& c) {
    return overlaps(out, bytes, c.lengths, 4ll * c.batch) || overlaps(out, bytes, c.table, 4ll * c.width, c.batch, 4ll * c.table_stride);
}

}  // namespace
}  // namespace kt

using namespace kt;

kt_status kt_paged_append(kt_ctx* ctx, const kt_paged_cache* cache, int32_t layer, const float* q, const float* k,
                          const float* v, int64_t q_stride, int64_t k_stride, int64_t v_stride, int32_t heads,
                          const float* inv_freq, int32_t rows_per_seq, const int32_t* counts, const int32_t* depths,
                          void* q_out, int32_t* status, void* stream) {
    if (!ctx) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (const char* why = check(cache)) return entry_fail(KT_ERR_INVALID_ARGUMENT, why);
    if (layer < 0 || layer >= cache->layers) return entry_fail(KT_ERR_INVALID_ARGUMENT, "layer out of range");
    if (rows_per_seq < 0) return entry_fail(KT_ERR_INVALID_ARGUMENT, "Negative row count");
    if (rows_per_seq == 0) return KT_OK;
    if (!k || !v || !inv_freq || (q && !q_out)) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (q ? heads < 1 || heads > 65535 : heads != 0)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "heads must be in 1..65535, or 0 without q");
    const int64_t width = static_cast<int64_t>(cache->kv_heads) * cache->head_dim;
    if (k_stride < width || v_stride < width || (q && q_stride < static_cast<int64_t>(heads) * cache->head_dim))
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows of q, k or v are shorter than their heads");
    if (q && reinterpret_cast<uintptr_t>(q_out) % 8 != 0) return entry_fail(KT_ERR_INVALID_ARGUMENT, "q_out must be 8-byte aligned");
    const int64_t rows = static_cast<int64_t>(cache->batch) * rows_per_seq;
    if (rows > (1ll << 31) - 1) return entry_fail(KT_ERR_INVALID_ARGUMENT, "too many rows");
    // (CTAs have parts of a row each, in no order)
    const auto read = [&](const void* out, int64_t bytes) {
        return overlaps(out, bytes, q, 4ll * heads * cache->head_dim, rows, 4 * q_stride) || overlaps(out, bytes, k, 4 * width, rows, 4 * k_stride) ||
               overlaps(out, bytes, v, 4 * width, rows, 4 * v_stride) || overlaps(out, bytes, inv_freq, 2ll * cache->head_dim) ||
               overlaps(out, bytes, counts, 4ll * cache->batch) || overlaps(out, bytes, depths, 4 * rows) || overlaps_places(out, bytes, *cache);
    };
    const int64_t q_bytes = q ? 2 * rows * heads * cache->head_dim : 0;
    if (read(q_out, q_bytes) || read(status, 4) || overlaps(status, 4, q_out, q_bytes))
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "q_out and status must not overlap each other or what the call reads");
    return c_entry(ctx, [&] {
        const auto quads = [](const float* p, int64_t stride) { return aligned16(p) && stride % 4 == 0; };
        const int aligned = (quads(q, q_stride) ? 1 : 0) | (quads(k, k_stride) ? 2 : 0) | (quads(v, v_stride) ? 4 : 0);
        const int at_once = kThreads / (cache->head_dim / 8), all = heads + 2 * cache->kv_heads;
        const int passes = (all + at_once - 1) / at_once;
        // A thread goes over several heads, for whom its sines are the same, where the rows fill the card.
        const int each = static_cast<int>(std::min<int64_t>(passes, std::max<int64_t>(1, rows * passes / (16ll * ctx->sm_count))));
        const Append a{q, k, v, inv_freq, counts, depths, q_out, status, q_stride, k_stride, v_stride, heads, rows_per_seq, layer, aligned, each};
        const dim3 grid(static_cast<unsigned>(rows), (passes + each - 1) / each);
        const auto kernel = cache->dtype == KT_BF16 ? paged_append_kernel<__nv_bfloat16> : paged_append_kernel<__half>;
        return entry_launch(launch_dependent(kernel, grid, dim3(kThreads), 0, static_cast<cudaStream_t>(stream), *cache, a),
                            "paged append launch");
    });
}

size_t kt_paged_scratch_bytes(kt_ctx* ctx) {
    return ctx ? kPagedPartsAt + std::max(paged_rows_bytes(), paged_many_bytes(ctx->sm_count)) : 0;
}

kt_status kt_paged_attention(kt_ctx* ctx, const kt_paged_cache* cache, int32_t layer, const void* q, int64_t q_stride,
                             void* out, int32_t out_dtype, int32_t rows_per_seq, const int32_t* counts,
                             const uint32_t* visible, int32_t heads, float scale, void* scratch, void* stream) {
    if (!ctx) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (const char* why = check(cache)) return entry_fail(KT_ERR_INVALID_ARGUMENT, why);
    if (layer < 0 || layer >= cache->layers) return entry_fail(KT_ERR_INVALID_ARGUMENT, "layer out of range");
    if (rows_per_seq < 0) return entry_fail(KT_ERR_INVALID_ARGUMENT, "Negative row count");
    if (rows_per_seq == 0) return KT_OK;
    if (!q || !out || !scratch) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (heads < 1 || heads > 65535 || heads % cache->kv_heads != 0)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "heads must be a positive multiple of kv_heads, at most 65535");
    if (q_stride < static_cast<int64_t>(heads) * cache->head_dim)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "rows of q are shorter than heads * head_dim");
    if (out_dtype != cache->dtype && out_dtype != KT_FP32)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "out_dtype must be the cache's or KT_FP32");
    const float factor = static_cast<float>(scale * 1.4426950408889634);
    if (!std::isfinite(factor)) return entry_fail(KT_ERR_INVALID_ARGUMENT, "scale must be finite, in powers of two as well");
    if (!aligned16(scratch)) return entry_fail(KT_ERR_INVALID_ARGUMENT, "scratch must be 16-byte aligned");
    if (visible && rows_per_seq > kMostNodes) return entry_fail(KT_ERR_INVALID_ARGUMENT, "visible needs at most 1024 rows a sequence");
    // (vectors of a sequence, and items of all, are counted in 32 bits)
    if (static_cast<int64_t>(rows_per_seq) * heads > (1 << 30) ||
        static_cast<int64_t>(rows_per_seq) * heads / cache->kv_heads * cache->batch > (1ll << 31) - 1)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "too many rows");
    // (a CTA writes the results of the queries that it has read, or that all who share them have: they may take their place)
    const int64_t rows = static_cast<int64_t>(cache->batch) * rows_per_seq, width = static_cast<int64_t>(heads) * cache->head_dim;
    const int64_t bytes = rows * width * (out_dtype == KT_FP32 ? 4 : 2);
    const bool in_place = out == q && (q_stride == width || rows == 1) && out_dtype == cache->dtype;
    if ((!in_place && overlaps(out, bytes, q, 2 * width, rows, 2 * q_stride)) || overlaps(out, bytes, counts, 4ll * cache->batch) ||
        overlaps(out, bytes, visible, 4 * rows * ((rows_per_seq + 31) / 32)) || overlaps_places(out, bytes, *cache))
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "out must not overlap what the call reads, but for the queries it takes the place of");
    return c_entry(ctx, [&] {
        PagedAttention a{};
        a.table = cache->table, a.lengths = cache->lengths, a.counts = counts, a.visible = visible;
        a.q = q, a.out = out, a.scratch = scratch, a.q_stride = q_stride;
        a.batch = cache->batch, a.kv_heads = cache->kv_heads, a.head_dim = cache->head_dim, a.pages = cache->pages;
        a.page_shift = cache->page == 16 ? 4 : cache->page == 32 ? 5 : cache->page == 64 ? 6 : 7;
        a.table_stride = cache->table_stride, a.capacity = cache->width * cache->page;
        a.rows = rows_per_seq, a.heads = heads, a.group = heads / cache->kv_heads, a.words = (rows_per_seq + 31) / 32;
        // (with a scale of 0 masked scores still have to be -inf, the others alike)
        a.factor = scale == 0.0f ? 1e-38f : factor;
        a.out_f32 = out_dtype == KT_FP32;
        a.aligned = (reinterpret_cast<uintptr_t>(q) % 16 == 0 && q_stride % 8 == 0 ? 1 : 0) | (aligned16(out) ? 2 : 0);
        return entry_launch(launch_paged_attention(*cache, layer, a, ctx->sm_count, ctx->d_error, static_cast<cudaStream_t>(stream)),
                            "paged attention launch");
    });
}

kt_status kt_paged_accept(kt_ctx* ctx, const kt_paged_cache* cache, const int32_t* tokens, const int32_t* parents,
                          const int32_t* choices, int32_t rows_per_seq, const int32_t* counts, int32_t* accepted,
                          int32_t* taken, int32_t* status, void* stream) {
    if (!ctx) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (const char* why = check(cache)) return entry_fail(KT_ERR_INVALID_ARGUMENT, why);
    if (!tokens || !parents || !choices || !accepted || !taken) return entry_fail(KT_ERR_INVALID_ARGUMENT, "NULL argument");
    if (rows_per_seq < 1 || rows_per_seq > kMostNodes)
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "a drafted tree has 1..1024 nodes");
    // (every CTA walks the trees for itself, while one already writes what it found)
    const int64_t nodes = 4ll * cache->batch * rows_per_seq, each = 4ll * cache->batch;
    const auto read = [&](const void* out, int64_t bytes) {
        return overlaps(out, bytes, tokens, nodes) || overlaps(out, bytes, parents, nodes) || overlaps(out, bytes, choices, nodes) ||
               overlaps(out, bytes, counts, each) || overlaps_places(out, bytes, *cache);
    };
    if (read(accepted, nodes) || read(taken, each) || read(status, 4) || overlaps(accepted, nodes, taken, each) ||
        overlaps(status, 4, accepted, nodes) || overlaps(status, 4, taken, each))
        return entry_fail(KT_ERR_INVALID_ARGUMENT, "accepted, taken and status must not overlap each other or what the call reads");
    return c_entry(ctx, [&] {
        const Accept a{tokens, parents, choices, counts, accepted, taken, status, rows_per_seq};
        return entry_launch(launch_dependent(paged_accept_kernel, dim3(2 * cache->layers, cache->batch), dim3(kThreads), 0,
                                             static_cast<cudaStream_t>(stream), *cache, a),
                            "paged accept launch");
    });
}
