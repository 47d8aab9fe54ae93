// kt_kv8_attention.cu -- attention over the 8-bit key/value cache.
//
// Row t of sequence b with n = lengths[b]: for each query head, over slots
// j <= n + t,  s_j = scale * (q . K_j),  out = sum_j softmax(s)_j V_j, with
// K_j = code * scale of the slot's block.
//
// Codes are whole numbers of at most 128, so the products run on tensor cores at
// fp32 accuracy once the fp32 operand is cut into terms that they take exactly.  The
// query becomes three signed bytes, 24 bits relative to its largest component, and its
// products with the keys' codes are integers, exact, with no conversion of the codes.
// The probabilities become two fp16 terms, x = hi + lo with hi = fp16(x) and
// lo = fp16(x - hi), 22 bits of each, and the values' codes are exact in fp16.  The
// scales of the blocks multiply the sums in fp32.
#include <cuda_fp16.h>

#include "kt_kv8.h"

namespace kt {
namespace {

constexpr int kWarps = 4;

// ------------------------------------------------------------ few query rows
//
// The query vectors that share a key/value head (rows_per_seq x heads / kv_heads
// of them) go eight to a tile: one m16n8k32 integer product holds their high bytes
// in rows 0..7 and their middle bytes in rows 8..15, a second their low bytes; the
// fp16 product of the probabilities holds hi terms in rows 0..7, lo terms in 8..15.
// So a thread finds all sums of a score in its own accumulators, and probabilities
// leave it in the layout the second product reads.  Work is the list of all tiles of
// kKeys slots over (sequence, key/value head, vector tile), cut into equal runs, one per
// CTA: ragged batches and single long sequences load every SM alike.  A warp takes
// every kWarps-th tile of its CTA's run through its own ring of asynchronous copies;
// nothing waits for another warp until an item's last tile, where the warps merge their
// maxima, sums and weighted sums.  Items cut between CTAs are merged by the last CTA to
// arrive, in the order of the cuts: equal bits on every run.
// Bound by memory at full batches, 64 sequences of 16k slots, 8 heads of 128: 445 us for
// 2.09 GB, 4.7 TB/s; one of 120001 slots 64 us, 3.9 TB/s; by latency when short: 301 slots of
// 2 heads of 64 6.7 us.  (With queries as two fp16 terms, which need the keys' codes
// converted, and one CTA of eight warps an SM: 507, 75 and 12 us.)

constexpr int kKeys = 32;
constexpr int kVectors = 8;
constexpr int kMostCtas = 456;  // of a launch
static_assert(kMostCtas <= kKv8MaxCtas, "a counter each");
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are kept 2^12 times larger, so that the fp16 terms of small ones
// stay clear of the subnormals; the factor cancels in the division by their sum.
constexpr float kLift = 12.0f;

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ float lds32(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
    return v;
}
// Asynchronous copies global -> shared.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// Bytes 0 and 2 of w, two codes, as an fp16 pair: with its sign bit flipped a code is
// 0x64xx = 1024 + 128 + code, less 1152 is the code.  (A mask and an exclusive or run
// at twice the rate of a byte permutation.)
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t w) {
    const uint32_t r = (w & 0x00ff00ffu) ^ 0x64806480u;
    return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&r), __half2half2(__ushort_as_half(0x6480))));
}
// Four floats of magnitude <= kQueryMax -> their nearest integers' signed digits to
// base 256, four to a word: high, middle, low.
constexpr float kQueryMax = 127.0f * 65536.0f + 127.0f * 256.0f + 127.0f;
__device__ __forceinline__ void three_bytes(const float (&x)[4], uint32_t& high, uint32_t& middle, uint32_t& low) {
    high = middle = low = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = __float2int_rn(x[i]);
        const int l = static_cast<int8_t>(n), rest = (n - l) >> 8, m = static_cast<int8_t>(rest), h = (rest - m) >> 8;
        low |= static_cast<uint32_t>(l & 255) << (8 * i);
        middle |= static_cast<uint32_t>(m & 255) << (8 * i);
        high |= static_cast<uint32_t>(h & 255) << (8 * i);
    }
}
// A thread's part of a query vector (four threads share one) as signed bytes in the
// layout of the first product; returns what a unit of the whole numbers is worth.
// Below 2^-100 a query counts as 0; where it is not finite every score is NaN.
template <int kSteps>
__device__ __forceinline__ float cut_query(float (&x)[2 * kSteps][4], uint32_t (&qa)[kSteps][6]) {
    uint32_t top = 0;  // the largest magnitude, by its bits: NaN above infinity
#pragma unroll
    for (int s = 0; s < 2 * kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[s][i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float largest = __uint_as_float(top);
    const float up = top < 0x0d800000u ? 0.0f : kQueryMax / largest;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[2 * s + i][j] = fminf(fmaxf(x[2 * s + i][j] * up, -kQueryMax), kQueryMax);
            three_bytes(x[2 * s + i], qa[s][2 * i], qa[s][2 * i + 1], qa[s][4 + i]);
        }
    return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : largest / kQueryMax;
}
// x0, x1 as their two fp16 terms, packed in pairs.
__device__ __forceinline__ void two_terms(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = h2_bits(h);
    lo = h2_bits(__floats2half2_rn(x0 - f.x, x1 - f.y));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A place in the list of work: tile `tile` of item `item` (key/value head times vector
// tile) of sequence b, whose items have `tiles` tiles each; the item starts at list
// index `base`.  An item counts as kStart tiles more than it has, ahead of its first:
// what a CTA spends on entering and leaving it.
struct Place {
    int64_t base;
    int b, item, tile, tiles;
};
// Quotients whose operands mostly fit 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

template <int HDP>
struct DecodeShape {
    static constexpr int kStages = 3;
    static constexpr int kStart = HDP == 128 ? 12 : 24;
    // Items up to this many tiles stay whole where there are CTAs enough: 4 tiles take 0.35 us of
    // head_dim 64, 0.8 of 128, joining the parts of an item 3.5 us (700 slots, 22 tiles, of
    // 2 heads x 64: whole 9.3 us, cut 10.7; of 8 heads x 128: whole 13.0, cut 11.9).
    static constexpr int kUncut = HDP == 128 ? 16 : 32;
    static constexpr int kTileBytes = kKeys * HDP;               // one of keys, values
    static constexpr int kStageBytes = 2 * kTileBytes + 16;      // and 2 + 2 scales
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kPartFloats = kVectors * (HDP + 2);     // sums, then maxima, then denominators
    static constexpr int kMeet = kWarps * kPartFloats > (kMostCtas + 2) * kVectors ? kWarps * kPartFloats : (kMostCtas + 2) * kVectors;
    static constexpr int kSmem = kWarps * kRing + kMeet * 4;
};

// Swizzle of 16-byte pieces that makes both fragment reads conflict-free: in
// 128-byte rows piece ^ ((row / 2 ^ (row & 1) * 2) % 4 * 2); 64-byte rows lie in
// pairs, (row & 1) * 4 + piece ^ (row / 2) % 4 * 2.
template <int HDP>
__device__ __forceinline__ int piece_offset(int row, int piece) {
    if (HDP == 128) return row * 128 + ((piece ^ ((((row >> 1) ^ ((row & 1) << 1)) & 3) << 1)) << 4);
    return (row >> 1) * 128 + ((((row & 1) * 4 + piece) ^ (((row >> 1) & 3) << 1)) << 4);
}

template <int HDP, bool kFine>
__global__ void __launch_bounds__(kWarps * 32) kv8_attention_kernel(Kv8Attention a, int vector_tiles, int aligned,
                                                                    float* __restrict__ parts,
                                                                    float* __restrict__ scores,
                                                                    float* __restrict__ lse) {
    using S = DecodeShape<HDP>;
    constexpr int kSteps = HDP / 32;       // k-steps of the first product
    constexpr int kPieces = HDP / 64;      // 16-byte pieces of a key a thread reads
    constexpr int kTiles = HDP / 8;        // n-tiles of the second product
    constexpr int kOwn = HDP / 4;          // dims of the output a thread holds
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int last_cta;
    const Kv8& c = a.cache;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, t = lane % 4, n8 = lane / 4;
    const int d = c.head_dim, pieces = d / 16, group = a.heads / c.kv_heads;
    const int vectors = a.rows_per_seq * group, items = c.kv_heads * vector_tiles;
    const uint32_t ring = dev::smem_u32(smem) + warp * S::kRing;
    float* const part_smem = reinterpret_cast<float*>(smem + kWarps * S::kRing);

    // Slots the rows of sequence b see, and tiles of one of its items.
    auto seen_by = [&](int b, int& rows) {
        rows = kv8_rows(a.counts, b, a.rows_per_seq);
        return rows == 0 ? 0 : min(kv8_held(c, b) + rows, c.capacity);
    };
    auto tiles_of = [&](int b) {
        int rows;
        return (seen_by(b, rows) + kKeys - 1) / kKeys;
    };
    if (a.counts != nullptr)  // rows that are no tokens
        for (int64_t r = blockIdx.x; r < static_cast<int64_t>(c.batch) * a.rows_per_seq; r += gridDim.x)
            if (static_cast<int>(r % a.rows_per_seq) >= kv8_rows(a.counts, static_cast<int>(r / a.rows_per_seq), a.rows_per_seq))
                for (int i = threadIdx.x; i < a.heads * d; i += blockDim.x) a.context[r * a.heads * d + i] = 0.0f;

    // This CTA's run [begin, end) of the list.
    int64_t real_tiles = 0, sequences = 0;
    int longest = 0;
    for (int b = lane; b < c.batch; b += 32) {
        const int n = tiles_of(b);
        real_tiles += n;
        longest = max(longest, n);
        sequences += n > 0;
    }
    for (int o = 16; o > 0; o >>= 1) {
        real_tiles += __shfl_xor_sync(0xffffffffu, real_tiles, o);
        sequences += __shfl_xor_sync(0xffffffffu, sequences, o);
        longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    }
    real_tiles *= items;
    const int64_t total = real_tiles + sequences * items * S::kStart;
    // A CTA an item, or one for each kWarps tiles of long ones, as far as the grid goes.  (One for
    // each 2 kWarps tiles left 15 items of one tile to one CTA: 65 us, now 6.8.)
    const int64_t whole = max(static_cast<int64_t>(1), sequences * items);
    const int64_t ctas = min(static_cast<int64_t>(gridDim.x),
                             longest <= S::kUncut ? whole : whole * max(static_cast<int64_t>(1), quotient(real_tiles, whole * kWarps)));
    if (blockIdx.x >= ctas) return;
    const int64_t share = quotient(total, ctas), spare = total - share * ctas;  // the first `spare` runs are one longer
    auto run_begin = [&](int64_t cta) { return cta * share + min(cta, spare); };
    auto cta_of = [&](int64_t i) {  // the CTA whose run holds list index i
        const int64_t longer = spare * (share + 1);
        return i < longer ? quotient(i, share + 1) : spare + quotient(i - longer, share);
    };
    const int64_t begin = run_begin(blockIdx.x), end = run_begin(blockIdx.x + 1);
    Place at{0, 0, 0, 0, 0};
    for (int b0 = 0; b0 < c.batch; b0 += 32) {
        const int mine = b0 + lane < c.batch ? tiles_of(b0 + lane) : 0;
        int64_t upto = mine > 0 ? static_cast<int64_t>(mine + S::kStart) * items : 0;
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t after = __ballot_sync(0xffffffffu, at.base + upto > begin);
        if (after != 0) {
            const int l = __ffs(after) - 1;
            at.b = b0 + l;
            at.tiles = __shfl_sync(0xffffffffu, mine, l);
            at.base += __shfl_sync(0xffffffffu, upto, l) - static_cast<int64_t>(at.tiles + S::kStart) * items;
            break;
        }
        at.base += __shfl_sync(0xffffffffu, upto, 31);
    }
    at.item = static_cast<int>(quotient(begin - at.base, at.tiles + S::kStart));
    at.base += static_cast<int64_t>(at.item) * (at.tiles + S::kStart);
    at.tile = static_cast<int>(max(static_cast<int64_t>(0), begin - at.base - S::kStart));

    // Where the run's tiles of p's item end, and whether the run goes on after the item.
    auto stop_of = [&](const Place& p) {
        return static_cast<int>(min(static_cast<int64_t>(p.tiles), max(static_cast<int64_t>(0), end - p.base - S::kStart)));
    };
    auto goes_on = [&](const Place& p) { return p.base + p.tiles + S::kStart < end; };
    // The first item after `p`'s: moves p to its tile 0.
    auto next_item = [&](Place& p) {
        p.base += p.tiles + S::kStart;
        p.tile = 0;
        if (++p.item < items) return;
        p.item = 0;
        do ++p.b;
        while (p.b < c.batch && (p.tiles = tiles_of(p.b)) == 0);
    };

    // The query of this thread's fragments at place p, ahead of its use and of the copies
    // that would delay it: dims 16 (t + 4 (s / 4)) + 4 (s % 4) ..
    float x[2 * kSteps][4];
    auto load_query = [&](const Place& p) {
        const int h = p.item / vector_tiles, vector = (p.item - h * vector_tiles) * kVectors + n8, row = vector / group;
        const bool real = vector < vectors && row < kv8_rows(a.counts, p.b, a.rows_per_seq);
        const float* q = a.q + (static_cast<int64_t>(p.b) * a.rows_per_seq + row) * a.q_stride +
                         static_cast<int64_t>(h * group + vector % group) * d;
#pragma unroll
        for (int s = 0; s < 2 * kSteps; ++s) {
            const int dim = 16 * (t + 4 * (s / 4)) + 4 * (s % 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[s][i] = 0.0f;
            if (real && dim < d) {
                if (aligned & 1) {
                    const float4 f = *reinterpret_cast<const float4*>(q + dim);
                    x[s][0] = f.x, x[s][1] = f.y, x[s][2] = f.z, x[s][3] = f.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[s][i] = q[dim + i];
                }
            }
        }
    };
    if (at.tile < stop_of(at)) load_query(at);

    // The warp's copies run ahead of its work over the same sequence of tiles.
    Place ahead = at;
    bool ahead_on = true;
    ahead.tile += warp;
    int fill = 0;
    // A lane copies piece `lane % kPieceCount` of every kCopyRows-th row.  Slots past the
    // last one seen come along (their scores are masked, their probabilities 0, and codes
    // are finite whatever they are); pieces past head_dim are left out, and what lies in
    // their place meets zeros of the query, or dims that nobody writes.
    constexpr int kPieceCount = HDP / 16, kCopyRows = 32 / kPieceCount, kCopies = kKeys / kCopyRows;
    const bool copies = lane % kPieceCount < pieces;
    const int64_t lane_from = static_cast<int64_t>(lane / kPieceCount) * d + lane % kPieceCount * 16;
    const uint32_t lane_to[2] = {static_cast<uint32_t>(piece_offset<HDP>(lane / kPieceCount, lane % kPieceCount)),
                                 static_cast<uint32_t>(piece_offset<HDP>(kCopyRows + lane / kPieceCount, lane % kPieceCount))};
    const int8_t *ahead_k, *ahead_v;  // of the lane, at slot 0 of the item
    const float* ahead_s;             // lanes 0, 1: the keys' scales, 2, 3: the values'
    auto enter = [&] {
        const int64_t head = static_cast<int64_t>(ahead.b) * c.kv_heads + ahead.item / vector_tiles;
        ahead_k = c.k_codes + head * c.capacity * d + lane_from;
        ahead_v = c.v_codes + head * c.capacity * d + lane_from;
        ahead_s = (lane < 2 ? c.k_scales : c.v_scales) + head * (c.capacity / c.block);
    };
    enter();
    const int block_shift = 31 - __clz(c.block);
    auto issue = [&] {
        while (ahead_on && ahead.tile >= stop_of(ahead)) {  // past items without a tile of this warp
            if ((ahead_on = goes_on(ahead))) {
                next_item(ahead);
                ahead.tile = warp;
                enter();
            }
        }
        if (ahead_on) {
            const int first = ahead.tile * kKeys;
            const uint32_t stage = ring + fill * S::kStageBytes;
            const int8_t* k = ahead_k + static_cast<int64_t>(first) * d;
            const int8_t* v = ahead_v + static_cast<int64_t>(first) * d;
            const bool all = first + kKeys <= c.capacity;  // else the first half of the tile
            if (copies) {
#pragma unroll
                for (int i = 0; i < kCopies; ++i) {
                    if (i >= kCopies / 2 && !all) break;
                    const uint32_t to = stage + lane_to[i & 1] + (i & ~1) * (kCopyRows * HDP);
                    copy16(to, k + i * kCopyRows * d);
                    copy16(to + S::kTileBytes, v + i * kCopyRows * d);
                }
            }
            if (lane < 4 && (all || !(lane & 1)))  // scales of slots first.. and first + 16..
                copy4(stage + 2 * S::kTileBytes + lane * 4, ahead_s + ((first + (lane & 1) * 16) >> block_shift));
            ahead.tile += kWarps;
        }
        copy_commit();
        fill = fill + 1 == S::kStages ? 0 : fill + 1;
    };
#pragma unroll
    for (int i = 0; i < S::kStages; ++i) issue();

    int use = 0;
    for (bool more = true; more;) {  // one segment: the run's tiles of one item
        const int stop = stop_of(at);
        more = goes_on(at);
        if (at.tile >= stop) break;  // the run ends ahead of the item's first tile
        int rows;
        const int seen = seen_by(at.b, rows), held = kv8_held(c, at.b);
        const int h = at.item / vector_tiles, vt = at.item - h * vector_tiles;
        const int vector = vt * kVectors + n8, row = vector / group;  // of this thread's fragments
        const bool real = vector < vectors && row < rows;
        const int limit = real ? min(held + row + 1, seen) : 0;                  // slots the vector sees
        const int64_t head = static_cast<int64_t>(at.b) * c.kv_heads + h;

        // Step s of the first product contracts the dims 16 (t + 4 (s / 2)) + 8 (s % 2) .. + 7 of
        // thread t: the words its 16-byte pieces of a key hold.
        uint32_t qa[kSteps][6];  // high, middle of the first four, of the last four; low of both
        const float factor = a.scale * kLog2e * cut_query<kSteps>(x, qa);
        float o[kOwn], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) o[i] = 0.0f;

        for (int tile = at.tile + warp; tile < stop; tile += kWarps) {
            copy_wait<S::kStages - 1>();
            __syncwarp();
            const uint32_t stage = ring + use * S::kStageBytes;
            const int first = tile * kKeys;
            float s[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int upper[4] = {0, 0, 0, 0}, lower[4] = {0, 0, 0, 0};
#pragma unroll
                for (int u = 0; u < kPieces; ++u) {
                    const uint4 w = lds128(stage + piece_offset<HDP>(8 * j + n8, t + 4 * u));
                    const uint32_t* const q0 = qa[2 * u];
                    const uint32_t* const q1 = qa[2 * u + 1];
                    mma(upper, q0[0], q0[1], q0[2], q0[3], w.x, w.y);
                    mma(lower, q0[4], 0, q0[5], 0, w.x, w.y);
                    mma(upper, q1[0], q1[1], q1[2], q1[3], w.z, w.w);
                    mma(lower, q1[4], 0, q1[5], 0, w.z, w.w);
                }
                // |middle sums| <= 128 x 128 x 128: 256 of them and a low sum stay below 2^30
                const float ks = lds32(stage + 2 * S::kTileBytes + (j >> 1) * 4) * factor;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    s[j][i] = fmaf(static_cast<float>(upper[i]), 65536.0f, static_cast<float>(upper[2 + i] * 256 + lower[i])) * ks;
            }
            if (first + kKeys > held + 1) {  // the first row's end, or the end of all, lies in this tile
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        if (first + 8 * j + 2 * t + i >= limit) s[j][i] = -INFINITY;
            }
            if (scores != nullptr && vector < vectors) {
                float* to = scores + (head * vectors + vector) * c.capacity + first;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (first + 8 * j < c.capacity)
                        *reinterpret_cast<float2*>(to + 8 * j + 2 * t) = make_float2(s[j][0], s[j][1]);
            }
            float top = m;
#pragma unroll
            for (int j = 0; j < 4; ++j) top = fmaxf(top, fmaxf(s[j][0], s[j][1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float from = (top == -INFINITY ? 0.0f : top) - kLift;
            if (__any_sync(0xffffffffu, top > m)) {
                const float fade = m == -INFINITY ? 0.0f : ex2((m - kLift) - from);
                l *= fade;
#pragma unroll
                for (int i = 0; i < kOwn; ++i) o[i] *= fade;
            }
            m = top;
            uint32_t pa[2][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p0 = ex2(s[j][0] - from), p1 = ex2(s[j][1] - from);
                l += p0 + p1;
                two_terms(p0, p1, pa[j >> 1][(j & 1) * 2], pa[j >> 1][(j & 1) * 2 + 1]);
            }
            // a block that the vector does not see has no scale, whatever is there
            const float vs0 = first < limit ? lds32(stage + 2 * S::kTileBytes + 8) : 0.0f;
            const float vs1 = first + 16 < limit ? lds32(stage + 2 * S::kTileBytes + 12) : 0.0f;
            // values: thread (t, n8) reads dims n8 * kTiles .. of slots 2t, 2t + 1, 2t + 8, 2t + 9 of
            // each 16; n-tile q of the product is dim n8 * kTiles + q
            uint32_t v[2][4][HDP / 32];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int slot = 16 * kk + 8 * (r >> 1) + 2 * t + (r & 1);
                    if (HDP == 128) {
                        const uint4 w = lds128(stage + S::kTileBytes + piece_offset<HDP>(slot, n8));
                        v[kk][r][0] = w.x, v[kk][r][1] = w.y, v[kk][r][HDP / 32 - 2] = w.z, v[kk][r][HDP / 32 - 1] = w.w;
                    } else {
                        const uint2 w = lds64(stage + S::kTileBytes + piece_offset<HDP>(slot, n8 >> 1) + (n8 & 1) * 8);
                        v[kk][r][0] = w.x, v[kk][r][1] = w.y;
                    }
                }
#pragma unroll
            for (int w = 0; w < HDP / 32; ++w) {
                float acc[4][4] = {};  // four n-tiles: bytes 0..3 of the words
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    uint32_t x[2], y[2];  // bytes 0, 1 and 2, 3 of two slots side by side
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        x[r] = dev::prmt(v[kk][2 * r][w], v[kk][2 * r + 1][w], 0x5410);
                        y[r] = dev::prmt(v[kk][2 * r][w], v[kk][2 * r + 1][w], 0x7632);
                    }
                    mma(acc[0], pa[kk], codes_to_half2(x[0]), codes_to_half2(x[1]));
                    mma(acc[1], pa[kk], codes_to_half2(x[0] >> 8), codes_to_half2(x[1] >> 8));
                    mma(acc[2], pa[kk], codes_to_half2(y[0]), codes_to_half2(y[1]));
                    mma(acc[3], pa[kk], codes_to_half2(y[0] >> 8), codes_to_half2(y[1] >> 8));
                    if (kFine || kk == 1) {  // blocks of 16 slots: each half has its own scale
                        const float vs = kFine && kk == 0 ? vs0 : kFine ? vs1 : vs0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            o[4 * w + i] = fmaf(vs, acc[i][0] + acc[i][2], o[4 * w + i]);
                            o[kTiles + 4 * w + i] = fmaf(vs, acc[i][1] + acc[i][3], o[kTiles + 4 * w + i]);
                            if (kFine) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
                        }
                    }
                }
            }
            __syncwarp();
            issue();
            use = use + 1 == S::kStages ? 0 : use + 1;
        }

        // The item's (or its cut's) end: the warps' parts meet in shared memory.
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        float* mine = part_smem + warp * S::kPartFloats;
#pragma unroll
        for (int i = 0; i < kOwn; i += 4)
            *reinterpret_cast<float4*>(mine + n8 * HDP + t * kOwn + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        if (t == 0) {
            mine[kVectors * HDP + n8] = m - kLift;  // what the sums are relative to
            mine[kVectors * HDP + kVectors + n8] = l;
        }
        Place next = at;
        if (more) {
            next_item(next);
            if (stop_of(next) > 0) load_query(next);
        }
        __syncthreads();
        const bool whole = at.tile == 0 && stop == at.tiles;
        const int slot = at.tile == 0 ? 1 : 0;
        float* part = parts + (static_cast<int64_t>(blockIdx.x) * 2 + slot) * S::kPartFloats;
        // a part's weight relative to the largest maximum; a part without slots has none
        auto weigh = [](float pm, float psum, float top) { return psum == 0.0f ? 0.0f : ex2(pm - top); };
        auto finish = [&](int vec, int dim, float4 y, float top, float sum) {
            const int idx = vt * kVectors + vec, r = idx / group;
            if (idx >= vectors || r >= rows || dim >= d) return;
            const float by = 1.0f / sum;
            float* to = a.context + (static_cast<int64_t>(at.b) * a.rows_per_seq + r) * a.heads * d +
                        static_cast<int64_t>(h * group + idx % group) * d + dim;
            if (aligned & 2) {
                *reinterpret_cast<float4*>(to) = make_float4(y.x * by, y.y * by, y.z * by, y.w * by);
            } else {
                to[0] = y.x * by, to[1] = y.y * by, to[2] = y.z * by, to[3] = y.w * by;
            }
            if (dim == 0 && lse != nullptr) lse[head * vectors + idx] = top + log2f(sum);
        };
        const int valid = min(kVectors, vectors - vt * kVectors);
        for (int e = threadIdx.x; e < valid * (HDP / 4); e += kWarps * 32) {
            const int vec = e / (HDP / 4), dim = e % (HDP / 4) * 4;
            float top = -INFINITY, sum = 0.0f;
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_smem[w * S::kPartFloats + kVectors * HDP + vec]);
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int w = 0; w < kWarps; ++w) {
                const float* p = part_smem + w * S::kPartFloats;
                const float psum = p[kVectors * HDP + kVectors + vec], by = weigh(p[kVectors * HDP + vec], psum, top);
                const float4 f = *reinterpret_cast<const float4*>(p + vec * HDP + dim);
                sum = fmaf(by, psum, sum);
                y.x = fmaf(by, f.x, y.x), y.y = fmaf(by, f.y, y.y), y.z = fmaf(by, f.z, y.z), y.w = fmaf(by, f.w, y.w);
            }
            if (whole) {
                finish(vec, dim, y, top, sum);
            } else {
                *reinterpret_cast<float4*>(part + vec * HDP + dim) = y;
                if (dim == 0) {
                    part[kVectors * HDP + vec] = top;
                    part[kVectors * HDP + kVectors + vec] = sum;
                }
            }
        }
        if (!whole) {
            // the CTAs that share the item: those whose runs hold its first .. last tile
            const int64_t c0 = cta_of(at.base + S::kStart), c1 = cta_of(at.base + S::kStart + at.tiles - 1);
            int32_t* counter = static_cast<int32_t*>(a.scratch) + c0;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) last_cta = dev::atomic_add_acq_rel(counter, 1) == static_cast<int>(c1 - c0);
            __syncthreads();
            if (last_cta) {
                __threadfence();
                const int n = static_cast<int>(c1 - c0) + 1;
                auto part_of = [&](int x) { return parts + ((c0 + x) * 2 + (x == 0 ? 1 : 0)) * S::kPartFloats; };
                // every part's weight in shared memory, a warp to a vector
                float* const totals = part_smem;               // largest reference, sum of each vector
                float* const weight = part_smem + 2 * kVectors;  // [part][vector]
                for (int v = warp; v < valid; v += kWarps) {
                    float top = -INFINITY, sum = 0.0f;
                    for (int x = lane; x < n; x += 32) {
                        const float m = __ldcg(part_of(x) + kVectors * HDP + v), psum = __ldcg(part_of(x) + kVectors * HDP + kVectors + v);
                        const float now = fmaxf(top, m);
                        sum = (sum == 0.0f ? 0.0f : sum * ex2(top - now)) + weigh(m, psum, now) * psum;
                        top = now;
                        weight[x * kVectors + v] = psum == 0.0f ? -INFINITY : m;
                    }
                    float all = top;
                    for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
                    sum = sum == 0.0f ? 0.0f : sum * ex2(top - all);
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) totals[2 * v] = all, totals[2 * v + 1] = sum;
                }
                __syncthreads();
                for (int e = threadIdx.x; e < valid * (HDP / 4); e += kWarps * 32) {
                    const int vec = e / (HDP / 4), dim = e % (HDP / 4) * 4;
                    const float top = totals[2 * vec];
                    const float* from = parts + c0 * 2 * S::kPartFloats + vec * HDP + dim;  // the first CTA's slot 1, the others' 0
                    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 16
                    for (int x = 0; x < n; ++x) {
                        const float m = weight[x * kVectors + vec], by = m == -INFINITY ? 0.0f : ex2(m - top);
                        const float4 f = __ldcg(reinterpret_cast<const float4*>(from + (x == 0 ? 1 : 2 * x) * S::kPartFloats));
                        y.x = fmaf(by, f.x, y.x), y.y = fmaf(by, f.y, y.y);
                        y.z = fmaf(by, f.z, y.z), y.w = fmaf(by, f.w, y.w);
                    }
                    finish(vec, dim, y, top, totals[2 * vec + 1]);
                }
                if (threadIdx.x == 0) *counter = 0;
            }
        }
        __syncthreads();  // the merge area and last_cta are free again

        at = next;
    }
}

// The weight of each slot where the rows are few, from the scores and row sums that the
// attention left: w_j += sum over vectors of 2^(s_j - lse).  Bound by latency where the
// scores are few and in L2: 16 sequences of 130 to 8190 slots, 32 heads over 8 (8.5 MB)
// 8.5 us beside 43 of their attention; by memory where they are many: 64 sequences of 16k
// (131 MB, written and read) 118 us beside 371.  (Adding in the attention would need the
// row sums before they are known.)
__global__ void __launch_bounds__(256) kv8_add_weights_kernel(Kv8Attention a, const float* __restrict__ scores,
                                                              const float* __restrict__ lse) {
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Kv8& c = a.cache;
    const int j = (blockIdx.x * 256 + threadIdx.x) * 4, h = blockIdx.y, b = blockIdx.z;
    const int rows = kv8_rows(a.counts, b, a.rows_per_seq), group = a.heads / c.kv_heads;
    const int held = kv8_held(c, b), n = rows == 0 ? 0 : min(held + rows, c.capacity);
    if (j >= n) return;
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    const int vectors = a.rows_per_seq * group;
    float w[4] = {};
#pragma unroll 4
    for (int i = 0; i < rows * group; ++i) {
        const float4 s = *reinterpret_cast<const float4*>(scores + (head * vectors + i) * c.capacity + j);
        const float z = lse[head * vectors + i];
        w[0] += ex2(s.x - z), w[1] += ex2(s.y - z), w[2] += ex2(s.z - z), w[3] += ex2(s.w - z);
    }
    float* to = c.weights + head * c.capacity + j;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (j + i < n) to[i] += w[i];
}

// The weight of each slot where the rows are many: w_j += sum over rows and heads of
// 2^(s_j - lse), the scores formed again from the codes, as in the first product above.
// First every query vector is cut into bytes, once, as the products read them, eight
// vectors to a tile: kCutWords x 512 bytes and an int4 a vector, {what a unit of its
// whole numbers is worth, its lse, the slots it sees}.
template <int HDP>
constexpr int kCutWords = 6 * HDP / 128;  // 16-byte words of a lane
size_t cut_bytes(int32_t head_dim) { return (head_dim > 64 ? kCutWords<128> : kCutWords<64>) * 512 + 8 * sizeof(int4); }
template <int HDP>
__global__ void __launch_bounds__(kWarps * 32) kv8_cut_kernel(Kv8Attention a, int aligned, const float* __restrict__ lse,
                                                              uint4* __restrict__ cut, int4* __restrict__ facts) {
    constexpr int kSteps = HDP / 32;
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Kv8& c = a.cache;
    const int lane = threadIdx.x % 32, t = lane % 4, n8 = lane / 4, h = blockIdx.y, b = blockIdx.z;
    const int d = c.head_dim, group = a.heads / c.kv_heads, tiles = (a.rows_per_seq * group + 7) / 8;
    const int rows = kv8_rows(a.counts, b, a.rows_per_seq), vectors = rows * group;
    const int tile = blockIdx.x * kWarps + threadIdx.x / 32;
    if (tile * 8 >= vectors) return;
    const int v = tile * 8 + n8, row = v / group, of = h * group + v - row * group;
    const int64_t r = static_cast<int64_t>(b) * a.rows_per_seq + row;
    const float* q = a.q + r * a.q_stride + static_cast<int64_t>(of) * d;
    float x[2 * kSteps][4];
#pragma unroll
    for (int s = 0; s < 2 * kSteps; ++s) {
        const int dim = 16 * (t + 4 * (s / 4)) + 4 * (s % 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[s][i] = 0.0f;
        if (v < vectors && dim < d) {
            if (aligned & 1) {
                const float4 f = *reinterpret_cast<const float4*>(q + dim);
                x[s][0] = f.x, x[s][1] = f.y, x[s][2] = f.z, x[s][3] = f.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[s][i] = q[dim + i];
            }
        }
    }
    uint32_t qa[kSteps][6];
    const float unit = a.scale * kLog2e * cut_query<kSteps>(x, qa);
    const int64_t at = (static_cast<int64_t>(b) * c.kv_heads + h) * tiles + tile;
#pragma unroll
    for (int i = 0; i < kCutWords<HDP>; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = qa[(4 * i + e) / 6][(4 * i + e) % 6];
        cut[(at * kCutWords<HDP> + i) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (t == 0) {
        const int held = kv8_held(c, b);
        const float less = v < vectors ? lse[r * a.heads + of] * kLog2e : 0.0f;
        facts[at * 8 + n8] = make_int4(__float_as_int(unit), __float_as_int(less),
                                       v < vectors ? min(held + row + 1, min(held + rows, c.capacity)) : 0, 0);
    }
}
// A CTA has kWeightSlots slots of one key/value head, 64 to a warp, whose codes stay in
// registers, and runs over the tiles of vectors that see them, the next one's bytes on
// their way; a cluster shares the tiles where there are few slots, and its first CTA adds
// up.  Sums are in a fixed order: equal bits on every run.  Bound by the integer
// products, 512 clocks of a scheduler's tensor core for 512 scores, which are under way
// in 63% of the cycles: 2 sequences x 509 rows x 32 heads over 3500 slots of 128 dims
// 171 us, 6000 rows over themselves 1.2 ms.  (A warp to a slot on the fp32 units took 30
// times as long; queries cut again by each CTA 486 us; three CTAs on an SM, whose
// registers spill, 189; two or eight n-tiles together 180.)
constexpr int kWeightSlots = 64 * kWarps;
template <int HDP>
__global__ void __launch_bounds__(kWarps * 32, 2) kv8_weights_kernel(Kv8Attention a, const uint4* __restrict__ cut,
                                                                     const int4* __restrict__ facts, int splits) {
    constexpr int kSteps = HDP / 32, kPieces = HDP / 64, kTogether = 4;  // n-tiles whose products do not wait for one another
    __shared__ float sums[kWeightSlots];
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Kv8& c = a.cache;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, t = lane % 4, n8 = lane / 4;
    const int split = blockIdx.x % splits, h = blockIdx.y, b = blockIdx.z;  // (`splits` CTAs are a cluster)
    const int d = c.head_dim, group = a.heads / c.kv_heads, tiles = (a.rows_per_seq * group + 7) / 8;
    const int rows = kv8_rows(a.counts, b, a.rows_per_seq), held = kv8_held(c, b);
    const int seen = rows == 0 ? 0 : min(held + rows, c.capacity);
    const int block_first = static_cast<int>(blockIdx.x / splits) * kWeightSlots, first = block_first + 64 * warp;
    if (block_first >= seen) return;  // as the whole cluster does
    const int64_t head = static_cast<int64_t>(b) * c.kv_heads + h;
    const int8_t* codes = c.k_codes + head * c.capacity * d;
    uint4 k[8][kPieces];
    float ks[4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int u = 0; u < kPieces; ++u) {
            const int slot = first + 8 * j + n8, dim = 16 * (t + 4 * u);
            k[j][u] = make_uint4(0, 0, 0, 0);
            if (slot < seen && dim < d) k[j][u] = *reinterpret_cast<const uint4*>(codes + static_cast<int64_t>(slot) * d + dim);
        }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        ks[j] = first + 16 * j < seen ? c.k_scales[head * (c.capacity / c.block) + (first + 16 * j) / c.block] : 0.0f;

    // vector v belongs to row v / group; the first that sees a slot of the CTA
    const int end = (rows * group + 7) / 8;
    int tile = max(0, block_first - held) * group / 8 + split;
    cut += head * tiles * kCutWords<HDP> * 32 + lane;
    facts += head * tiles * 8 + n8;
    uint4 next[kCutWords<HDP>];
    int4 next_facts = make_int4(0, 0, 0, 0);
    auto load = [&](int x) {
#pragma unroll
        for (int i = 0; i < kCutWords<HDP>; ++i) next[i] = cut[(static_cast<int64_t>(x) * kCutWords<HDP> + i) * 32];
        next_facts = facts[static_cast<int64_t>(x) * 8];
    };
    float sum[8][2] = {};
    if (tile < end) load(tile);
#pragma unroll 1
    for (; tile < end; tile += splits) {
        uint32_t qa[kSteps][6];
#pragma unroll
        for (int i = 0; i < kCutWords<HDP>; ++i) {
            const uint32_t words[4] = {next[i].x, next[i].y, next[i].z, next[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) qa[(4 * i + e) / 6][(4 * i + e) % 6] = words[e];
        }
        const float unit = __int_as_float(next_facts.x), less = __int_as_float(next_facts.y);
        const int limit = next_facts.z;
        if (tile + splits < end) load(tile + splits);
        const bool part = __any_sync(0xffffffffu, limit < first + 64);  // some vector does not see all of the slots
#pragma unroll
        for (int j0 = 0; j0 < 8; j0 += kTogether) {
            int upper[kTogether][4] = {}, lower[kTogether][4] = {};
#pragma unroll
            for (int u = 0; u < 2 * kPieces; ++u)
#pragma unroll
                for (int j = 0; j < kTogether; ++j) {
                    const uint32_t* const q = qa[u];
                    const uint4 w4 = k[j0 + j][u / 2];
                    mma(upper[j], q[0], q[1], q[2], q[3], u % 2 ? w4.z : w4.x, u % 2 ? w4.w : w4.y);
                    mma(lower[j], q[4], 0, q[5], 0, u % 2 ? w4.z : w4.x, u % 2 ? w4.w : w4.y);
                }
#pragma unroll
            for (int j = 0; j < kTogether; ++j) {
                const float by = ks[(j0 + j) / 2] * unit;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float dot = fmaf(static_cast<float>(upper[j][i]), 65536.0f,
                                           static_cast<float>(upper[j][2 + i] * 256 + lower[j][i]));
                    float p = ex2(dot * by - less);
                    if (part && first + 8 * (j0 + j) + 2 * t + i >= limit) p = 0.0f;
                    sum[j0 + j][i] += p;
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            for (int o = 4; o < 32; o <<= 1) sum[j][i] += __shfl_xor_sync(0xffffffffu, sum[j][i], o);
            if (n8 == 0) sums[64 * warp + 8 * j + 2 * t + i] = sum[j][i];
        }
    dev::cluster_sync();
    if (split == 0)
        for (int i = threadIdx.x; i < min(kWeightSlots, seen - block_first); i += kWarps * 32) {
            float all = 0.0f;
            for (int x = 0; x < splits; ++x) {
                uint32_t at;
                float f;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(dev::smem_u32(sums + i)), "r"(x));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(at));
                all += f;
            }
            c.weights[head * c.capacity + block_first + i] += all;
        }
    dev::cluster_sync();  // nobody leaves while its sums are read
}

template <int HDP>
cudaError_t launch_weights(const Kv8Attention& a, int sm_count, int aligned, const float* lse, void* room, cudaStream_t s) {
    const Kv8& c = a.cache;
    const int tiles = (a.rows_per_seq * (a.heads / c.kv_heads) + 7) / 8;
    int4* facts = static_cast<int4*>(room);
    uint4* cut = reinterpret_cast<uint4*>(facts + static_cast<int64_t>(c.batch) * c.kv_heads * tiles * 8);
    cudaError_t e = launch_dependent(kv8_cut_kernel<HDP>, dim3((tiles + kWarps - 1) / kWarps, c.kv_heads, c.batch),
                                     dim3(kWarps * 32), 0, s, a, aligned, lse, cut, facts);
    if (e != cudaSuccess) return e;
    const int64_t blocks = (c.capacity + kWeightSlots - 1) / kWeightSlots, alone = blocks * c.kv_heads * c.batch;
    int splits = 1;  // while SMs lack a second CTA and there are tiles for more
    while (splits < 8 && alone * splits < 2 * sm_count && splits * 8 < tiles) splits *= 2;
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(static_cast<unsigned>(blocks * splits), c.kv_heads, c.batch);
    lc.blockDim = dim3(kWarps * 32);
    lc.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 2;
    return cudaLaunchKernelEx(&lc, kv8_weights_kernel<HDP>, a, static_cast<const uint4*>(cut), static_cast<const int4*>(facts), splits);
}

}  // namespace

namespace {
// Which kernel is the faster.  The one of this file reads the cache for every eight
// query vectors and spreads all tiles of 32 slots over the card: 1.3 ns a tile, with
// head_dim 128 and the codes in L2.  The one on tcgen05 gives 128 vectors to a CTA: 2 us
// for 128 slots of a wave of 148, or of their part where fewer share the slots out.
// (30 rows of 32 heads over 8, one sequence of 30000 slots: 171 us here, 55 there; 17
// rows, 2000 slots: 23 us here, 25 there.)  Smaller head_dims go by the same numbers, which
// keep this file's kernel too short there: 1 sequence of 500 slots, 14 heads over 2 of 64,
// 16 rows: 11.7 us here, 16.1 there, and there it runs.
// Both grow with the lengths, which only the device knows and which drop out:
//   sequences x kv_heads x eights x 4 x 1.3 ns  against  waves x 2 us.
// (The choice must not ask whether weights are accumulated: a context has the same bits
// either way.)
bool use_tiles(int64_t batch, int32_t rows_per_seq, int32_t heads, int32_t kv_heads) {
    const int64_t vectors = static_cast<int64_t>(rows_per_seq) * (heads / kv_heads);
    const int64_t eights = (vectors + 7) / 8, ctas = batch * kv_heads * ((vectors + 127) / 128);
    const double waves = ctas < kPromptCtas ? static_cast<double>(ctas) / kPromptCtas : static_cast<double>((ctas + kPromptCtas - 1) / kPromptCtas);
    return eights == 1 || static_cast<double>(batch * kv_heads * eights) * 5.2 < 2000.0 * waves;
}
int tiles_of_vectors(int32_t rows_per_seq, int32_t heads, int32_t kv_heads) {
    return (rows_per_seq * (heads / kv_heads) + kVectors - 1) / kVectors;
}
size_t round256(size_t n) { return (n + 255) / 256 * 256; }
size_t part_bytes(int32_t head_dim) {
    const size_t hdp = head_dim <= 64 ? 64 : 128;
    return round256(static_cast<size_t>(kKv8MaxCtas) * 2 * kVectors * (hdp + 2) * sizeof(float));
}
size_t lse_bytes(int32_t batch, int32_t rows_per_seq, int32_t heads) {
    return round256(static_cast<size_t>(batch) * rows_per_seq * heads * sizeof(float));
}

template <int HDP, bool kFine>
cudaError_t launch_tiles(const Kv8Attention& a, int sm_count, int aligned, float* parts, float* scores, float* lse,
                         cudaStream_t s) {
    using S = DecodeShape<HDP>;
    const auto kernel = kv8_attention_kernel<HDP, kFine>;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = allow_shared(kernel, S::kSmem, allowed);
    if (e != cudaSuccess) return e;
    const Kv8& c = a.cache;
    const int vt = tiles_of_vectors(a.rows_per_seq, a.heads, c.kv_heads);
    const int per_sm = 233472 / (S::kSmem + 1152);  // what shared memory holds
    // A CTA an item, or one for each kWarps tiles.
    const int64_t items = static_cast<int64_t>(c.batch) * c.kv_heads * vt, most = items * ((c.capacity + kKeys - 1) / kKeys);
    const int grid = static_cast<int>(std::min<int64_t>(std::min(sm_count * per_sm, kMostCtas),
                                                        std::max(items, most / kWarps)));
    return launch_dependent(kernel, dim3(grid), dim3(kWarps * 32), S::kSmem, s, a, vt, aligned, parts, scores, lse);
}
}  // namespace

size_t kv8_attention_bytes(int32_t batch, int32_t rows_per_seq, int32_t heads, int32_t kv_heads, int32_t head_dim,
                           int32_t capacity, bool weights) {
    size_t n = std::max(part_bytes(head_dim), round256(kv8_prompt_bytes(head_dim))) + lse_bytes(batch, rows_per_seq, heads);
    if (weights && use_tiles(batch, rows_per_seq, heads, kv_heads))
        n += static_cast<size_t>(batch) * rows_per_seq * heads * capacity * sizeof(float);
    else if (weights)
        n += static_cast<size_t>(batch) * kv_heads * tiles_of_vectors(rows_per_seq, heads, kv_heads) * cut_bytes(head_dim);
    return n;
}

cudaError_t launch_kv8_attention(const Kv8Attention& a, int sm_count, int32_t* err, cudaStream_t s) {
    const Kv8& c = a.cache;
    char* free = static_cast<char*>(a.scratch) + kKv8CounterBytes;
    float* parts = reinterpret_cast<float*>(free);
    const size_t lse_at = std::max(part_bytes(c.head_dim), round256(kv8_prompt_bytes(c.head_dim)));
    float* lse = reinterpret_cast<float*>(free + lse_at);
    const auto ok16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const int aligned = (ok16(a.q) && a.q_stride % 4 == 0 ? 1 : 0) | (ok16(a.context) ? 2 : 0);
    if (use_tiles(c.batch, a.rows_per_seq, a.heads, c.kv_heads)) {
        float* scores = reinterpret_cast<float*>(free + lse_at + lse_bytes(c.batch, a.rows_per_seq, a.heads));
        if (!a.accumulate) scores = nullptr;
        const bool fine = c.block == 16, wide = c.head_dim > 64;
        cudaError_t e = wide ? fine ? launch_tiles<128, true>(a, sm_count, aligned, parts, scores, lse, s)
                                    : launch_tiles<128, false>(a, sm_count, aligned, parts, scores, lse, s)
                        : fine ? launch_tiles<64, true>(a, sm_count, aligned, parts, scores, lse, s)
                               : launch_tiles<64, false>(a, sm_count, aligned, parts, scores, lse, s);
        if (e == cudaSuccess && a.accumulate)
            e = launch_dependent(kv8_add_weights_kernel, dim3((c.capacity + 1023) / 1024, c.kv_heads, c.batch), dim3(256),
                                 0, s, a, static_cast<const float*>(scores), static_cast<const float*>(lse));
        return e;
    }
    cudaError_t e = launch_kv8_prompt(a, aligned, parts, a.accumulate ? lse : nullptr, err, s);
    if (e == cudaSuccess && a.accumulate) {
        void* room = free + lse_at + lse_bytes(c.batch, a.rows_per_seq, a.heads);
        e = c.head_dim > 64 ? launch_weights<128>(a, sm_count, aligned, lse, room, s)
                            : launch_weights<64>(a, sm_count, aligned, lse, room, s);
    }
    return e;
}

}  // namespace kt
