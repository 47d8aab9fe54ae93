// kt_paged_many.cu -- attention over the paged 16-bit key/value cache for many query
// vectors a key/value head (drafted trees, prompts) on the 5th-generation tensor cores.
//
// 256 query vectors that share a key/value head are an item, over tiles of 128 slots whose
// keys and values pass through a ring of shared memory (boxes of pages by TMA).  Two
// streams of four warps have 128 vectors each, a lane of tensor memory and a thread to a
// vector; with 128 vectors or fewer, both have the same and every other tile, and are
// added at the end.  A stream works by halves of a tile, 64 slots:
//   S = Q K^T       tcgen05.mma, Q and K in shared memory, S in tensor memory
//   P = 2^(S * factor - reference), rounded to the cache's type, into S's own columns
//   O += P V        tcgen05.mma, P and O in tensor memory
// and while its softmax has one half, its issuing warp has the products of the other: P V of
// a half, then Q K^T of the same half of the next tile.  (Whole tiles, one set of scores a
// stream: products and softmax took turns, 4700 clocks a tile where halves took 3700, before a
// warp of its own waited for copies, with which halves take 3000 and whole tiles were not
// tried.)  The streams take turns with their powers of two, which one unit serves: left alone they fell
// into step and both waited for it, then both for the tensor cores.
//
// The reference of a vector is its largest score so far, less up to 2^8: only when a score
// passes it by more do O and the sum go over to a new one, which needs the products under
// way to end.  So the largest probability is rounded like the others.  Where few count, as in
// the cases below, results are off by 2.2e-3 of their size in bfloat16 and 2.7e-4 in fp16;
// always at the largest score by 1.8e-3 and 2.2e-4 (of which 1.7e-3 and 2.1e-4 are the result's
// own rounding), but then the prompt takes 189 us, the chunk 80, the trees 46.  The sum is of
// the probabilities before their rounding: a result is off by at most half a step of its sum
// of |p v|, of rounded ones by up to a whole step, though the 2.2e-3 would be 2.0e-3.  Sums,
// references and O are fp32.
//
// Masks.  Only tiles that some vector does not see in full (the last ones, and all that hold
// new tokens of a tree) look at them.  There values are read first: rows of the tile past the
// last slot and values that are not finite become zeros, and vectors that see one of the
// latter get NaN in its dim at their item's end; so nothing that is not seen reaches a result.
//
// Bound by the streams' turns with their powers of two, 750 clocks a half (512 of the unit),
// which the products just follow (2560 clocks of a tile's 3000: scores of 64 slots read the
// queries again, 48 clocks a step where 128 slots would take 64); and by what an item costs:
// about 5000 clocks to enter, 5500 to leave, and twice a tile for one with masks.  A prompt
// of 4093 rows of 32 heads over 8 of 128: 162 us, 847 TFLOP/s (141 back to back); 2 x 509 rows over 1000 to
// 2999 tokens 65 us; 4 trees of 63 rows over 2500 to 6001 tokens 40 us, about 6 of them the merge.
// (Some of the powers as polynomials on the fp32 units: 1 % faster with one in eight, 5 % slower with three.)
#include <algorithm>

#include "kt_paged.h"

namespace kt {
namespace {

using namespace paged;

constexpr int kLanes = 128;                // vectors of a stream (the MMA's M)
constexpr int kVectors = 2 * kLanes;       // of an item
constexpr int kTile = 128;                 // slots of a tile
// What entering an item costs, in tiles (a prompt of 4093 rows, cut: 157 us, counted as two 212, as six 162), the
// tiles that are worth a CTA, and up to how many an item is not cut (a tree of 20 rows over 300 tokens of each of 8
// sequences: 17.9 us, cut 19.3); from how many items to a CTA a prompt's are dealt whole (157 us cut, 141 dealt).
constexpr int kStart = 4, kLeast = 2, kWhole = 4, kDeal = 3;
constexpr int kIssueWarp = 8, kCopyWarp = 10, kLandWarp = 11;  // after the softmax warps; an issuing warp for each stream
constexpr int kThreads = 384;
constexpr float kLift = 6.0f;   // probabilities are 2^kLift times larger: fp16 keeps them to 2^-30 of the reference
constexpr float kSlack = 8.0f;   // the reference moves when a score passes it by this much (2^14 < fp16's largest)

template <int HDP>
struct ManyShape {
    static constexpr int kBlocks = HDP / 64;             // blocks of 64 dims: swizzled rows of 128 bytes
    static constexpr int kUnit = kBlocks * kTile * 128;  // queries of a stream; keys or values of a tile
    static constexpr int kRing = 2 * kUnit, kUnits = 4 * 128 / HDP;  // keys, values, keys, ...
    static constexpr int kBad = kRing + kUnits * kUnit;  // slots of an edge tile whose values are not finite: [2][3][4] words
    static constexpr int kStats = kBad + 128;            // of the second stream's vectors
    static constexpr int kWords = HDP / 32;              // of a bit for each dim
    static constexpr int kMap = kStats + 2 * kLanes * 4; // which dims of those slots: [2][2][slot][word]
    static constexpr int kMarks = kMap + 4 * kTile * kWords * 4;  // dims in which a vector gets NaN: [word][thread]
    static constexpr int kBars = kMarks + kWords * 256 * 4;
    static constexpr int kSmem = 1024 + kBars + 16 * kUnits + 14 * 8;
    static constexpr int kPart = kVectors * (HDP + 2);   // floats of a part: [HDP / 4][vector][4], references, sums
    static constexpr uint32_t kO = 256;                  // tensor memory: scores (then P) of stream x at 128 x, its O
    static_assert(kSmem <= 232448 && kO + 2 * HDP <= 512, "memories");
};

// An item that its CTA begins and later ones go on with, left for the merge.
struct Cut {
    int32_t parts, b, head, v0, valid, unused[3];
};
static_assert(sizeof(Cut) * kPagedManyCtas <= kPagedCutBytes, "a place each");

// Shared-memory descriptors, the low words (the issuing thread adds to 32 bits, not 64):
// 128-byte swizzle, atoms of 8 rows 1024 bytes apart, descriptor version 1.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_of(uint32_t addr, uint32_t lead) { return (addr & 0x3FFFFu) >> 4 | lead >> 4 << 16; }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Columns of this warp's 32 lanes, complete on return.  (One statement: between a load and
// its wait the compiler may copy the registers, which do not hold the values yet.)
__device__ __forceinline__ void ld(uint32_t addr, float (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
          "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
          "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
          "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31]),
          "=f"(r[32]), "=f"(r[33]), "=f"(r[34]), "=f"(r[35]), "=f"(r[36]), "=f"(r[37]), "=f"(r[38]), "=f"(r[39]),
          "=f"(r[40]), "=f"(r[41]), "=f"(r[42]), "=f"(r[43]), "=f"(r[44]), "=f"(r[45]), "=f"(r[46]), "=f"(r[47]),
          "=f"(r[48]), "=f"(r[49]), "=f"(r[50]), "=f"(r[51]), "=f"(r[52]), "=f"(r[53]), "=f"(r[54]), "=f"(r[55]),
          "=f"(r[56]), "=f"(r[57]), "=f"(r[58]), "=f"(r[59]), "=f"(r[60]), "=f"(r[61]), "=f"(r[62]), "=f"(r[63])
        : "r"(addr)
        : "memory");
}
// The same for 16 columns, complete on return.
__device__ __forceinline__ void ld16(uint32_t addr, float (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
          "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// Two fp32 operations at a time.
__device__ __forceinline__ uint64_t pair(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ bool bar_any(int id, int threads, bool mine) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all) : "r"(static_cast<uint32_t>(mine)), "r"(id), "r"(threads) : "memory");
    return all != 0;
}

// 64 scores of a vector to P in tensor memory; their sum.
template <typename T>
__device__ __forceinline__ float probabilities(const float (&s)[64], uint64_t by, uint64_t off, uint32_t p_tm) {
    uint64_t total[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 64; i += 32) {
        uint32_t p[16];
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
            float z0, z1;
            unpair(fma2(pair(s[i + j], s[i + j + 1]), by, off), z0, z1);
            z0 = ex2(z0), z1 = ex2(z1);
            total[j / 2 % 2] = add2(total[j / 2 % 2], pair(z0, z1));
            p[j / 2] = Half16<T>::pack(z0, z1);
        }
        st16(p_tm + i / 2, p);
    }
    float t0, t1;
    unpair(add2(total[0], total[1]), t0, t1);
    return t0 + t1;
}

template <typename T, int HDP>
__global__ void __launch_bounds__(kThreads, 1) paged_many_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                 const __grid_constant__ CUtensorMap v_map,
                                                                 const __grid_constant__ PagedAttention a,
                                                                 int32_t* __restrict__ err) {
    using S = ManyShape<HDP>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ uint32_t tmem_slot;
    const uint32_t raw = dev::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    unsigned char* const smem = smem_raw + (base - raw);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, d = a.head_dim;
    const uint32_t bars = base + S::kBars;
    auto full = [&](int x) { return bars + 16 * x; };
    auto empty = [&](int x) { return bars + 16 * x + 8; };
    // of stream x, for each half of a tile
    auto s_full = [&](int x, int half) { return bars + 16 * S::kUnits + 16 * x + 8 * half; };
    auto p_full = [&](int x, int half) { return s_full(x, half) + 32; };
    auto o_done = [&](int x, int half) { return s_full(x, half) + 64; };
    const uint32_t q_full = bars + 16 * S::kUnits + 96, finished = q_full + 8;
    Cut* const cuts = reinterpret_cast<Cut*>(static_cast<char*>(a.scratch) + kPagedCounterBytes);
    if (threadIdx.x == 0) {
        for (int x = 0; x < S::kUnits; ++x) {
            dev::mbar_init(full(x), 1);
            dev::mbar_init(empty(x), 2);  // an issuing warp each
        }
        for (int i = 0; i < 4; ++i) {
            dev::mbar_init(s_full(i / 2, i % 2), 1);
            dev::mbar_init(p_full(i / 2, i % 2), i % 2 ? 4 : 5);  // the softmax warps, and the landing one before a tile
            dev::mbar_init(o_done(i / 2, i % 2), 1);
        }
        dev::mbar_init(q_full, 11);  // the softmax warps, the landing one, and the issuing ones, which see every phase that way
        dev::mbar_init(finished, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        dev::prefetch_map(&k_map);
        dev::prefetch_map(&v_map);
    }
    dev::pdl_wait();
    if (threadIdx.x == 0) cuts[blockIdx.x].parts = 0;
    __shared__ Plan<kThreads / 32> plan;
    const WorkList<kThreads / 32, kVectors, kTile, kStart, kLeast, kWhole, kDeal> work{a, plan};
    if (!work.start()) {  // (its barriers also publish the mbarriers)
        dev::pdl_launch_dependents();
        if (warp == kCopyWarp) zero_rows(a);
        return;
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dev::smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = tmem_slot;
    const Item& it = plan.at[warp];
    // only now: a dependent kernel's CTA on this SM must not take the tensor memory first
    dev::pdl_launch_dependents();
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {  // a lane that has given up goes on without waiting
        if (ok && !wait_counted(bar, parity)) ok = false;
    };

    // An item of more than kLanes vectors has two streams over the same tiles, each with its vectors; one of fewer
    // has two over every other tile, with the same vectors, whose results are added at its end.
    if (warp < kIssueWarp) {
        const int x = warp / 4, row = threadIdx.x % kLanes;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(warp % 4) << 21), s_tm = lanes + kLanes * x, o_tm = lanes + S::kO + HDP * x;
        uint32_t* const bad_words = reinterpret_cast<uint32_t*>(smem + S::kBad);
        uint32_t* const marks = reinterpret_cast<uint32_t*>(smem + S::kMarks) + threadIdx.x;
        float* const parts = reinterpret_cast<float*>(static_cast<char*>(a.scratch) + kPagedPartsAt);
        const float factor = fabsf(a.factor);
        if (x == 1) bar_arrive(4, 256);  // the first stream has the first turn
        int64_t unit0 = 0;  // of the run's first tile of this item
        uint32_t done = 0;  // tiles of this stream
        do {
            const int from = it.from, to = it.to;
            if (from >= to) continue;
            const bool twice = it.valid > kLanes;
            const int step = twice ? 1 : 2, v = (twice ? kLanes * x : 0) + row;  // the vector of this thread, in the item
            bar_sync(1, 256);  // nobody works on the item before
            if (threadIdx.x < 24) bad_words[threadIdx.x] = 0;
#pragma unroll
            for (int w = 0; w < S::kWords; ++w) marks[256 * w] = 0;
            // Queries, 32 rows of this stream's, or half of them where both streams work on the same; lanes on neighbouring
            // pieces of a row
            {
                constexpr int kPieces = HDP / 8, kRows = 32 / kPieces;  // of 8 dims; rows at a time
                const int first = v - lane, c = lane % kPieces, valid = it.valid;
                const uint32_t to_q = base + (twice ? x * S::kUnit : 0) + c / 8 * (kTile * 128);
                const int64_t mine = v < valid ? place_of(a, it.b, it.head, it.v0 + v, a.q_stride) : 0;
                const uint16_t* const q = static_cast<const uint16_t*>(a.q);
                const bool aligned = a.aligned & 1;
#pragma unroll 1
                for (int half = twice ? 0 : x; half < (twice ? 2 : x + 1); ++half) {
#pragma unroll
                    for (int i = 0; i < kPieces / 2; ++i) {
                        const int r = half * 16 + i * kRows + lane / kPieces, line = row - lane + r;
                        const int64_t from_q = __shfl_sync(0xffffffffu, mine, r) + 8 * c;
                        const uint32_t at = to_q + line * 128 + ((c % 8 ^ (line & 7)) << 4);
                        const bool here = first + r < valid && 8 * c < d;
                        if (aligned) {
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(q + (here ? from_q : 0)), "r"(here ? 16 : 0));
                        } else {
                            uint32_t e[4] = {};
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (here) e[j] = q[from_q + 2 * j] | static_cast<uint32_t>(q[from_q + 2 * j + 1]) << 16;
                            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(e[0]), "r"(e[1]), "r"(e[2]), "r"(e[3]));
                        }
                    }
                }
            }
            bool no_page = false;
            for (int p = (from * kTile >> a.page_shift) + threadIdx.x; p <= (min(to * kTile, it.sees) - 1) >> a.page_shift; p += 256) {
                const int page = a.table[static_cast<int64_t>(it.b) * a.table_stride + p];
                no_page = no_page || page < 0 || page >= a.pages;
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            no_page = bar_any(1, 256, no_page);
            if (lane == 0) dev::mbar_arrive(q_full);

            // slots that all of the item's vectors see
            const int clear = no_page ? 0 : a.visible ? it.held : min(it.held + it.v0 / a.group + 1, it.sees);
            const int t = v < it.valid ? (it.v0 + v) / a.group : -1;
            const bool works = it.valid > v - lane;  // some vector of the warp
            float ref = -INFINITY, sum = 0.0f;
            int n = 0;  // tiles of this item
            for (int tile = from + (twice ? 0 : x); tile < to; tile += step, ++n, ++done) {
                const int slot = tile * kTile;
                const bool edge = slot + kTile > clear;
                const int group = twice ? 0 : x;
                uint32_t* const words = bad_words + 12 * group + 4 * (n % 3);
                uint32_t* const map = reinterpret_cast<uint32_t*>(smem + S::kMap) + (2 * group + n % 2) * (kTile * S::kWords);
                if (edge) {
                    // Values of slots past the last one seen count nothing, whatever is there, and values that are not
                    // finite count for the vectors that see them alone, who get NaN in their dims: zeros take their place.
                    const int cleaners = twice ? 256 : 128, me = twice ? static_cast<int>(threadIdx.x) : row, sees = it.sees;
                    const int64_t vu = unit0 + 2 * (tile - from) + 1;
                    // (the scores were issued after the values that lay in this place before had landed: the phase is no older one)
                    wait(s_full(x, 0), done & 1);
                    wait(full(static_cast<int>(vu % S::kUnits)), (vu / S::kUnits) & 1);
                    __syncwarp();
                    for (int e = me; e < kTile * S::kBlocks; e += cleaners) {
                        const int at = slot + e % kTile;
                        if (at < clear) continue;  // seen by all
                        uint4* const line = reinterpret_cast<uint4*>(smem + S::kRing + static_cast<uint32_t>(vu % S::kUnits) * S::kUnit + e * 128);
                        if (at >= sees || (no_page && !has_page(a, it.b, at))) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) line[i ^ (lane & 7)] = make_uint4(0, 0, 0, 0);
                            continue;
                        }
                        uint32_t over = 0, low = 0, high = 0;  // bits of the dims
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint4 w = line[i ^ (lane & 7)];
                            over |= not_finite<T>(w.x) | not_finite<T>(w.y) | not_finite<T>(w.z) | not_finite<T>(w.w);
                        }
                        if (over != 0) [[unlikely]] {
                            atomicOr(words + e % kTile / 32, 1u << (e % 32));
#pragma unroll 1
                            for (int i = 0; i < 32; ++i) {  // pairs of dims
                                uint32_t& w = reinterpret_cast<uint32_t*>(line + (i / 4 ^ (lane & 7)))[i % 4];
                                const uint32_t bad = not_finite<T>(w);
                                const uint32_t two = (bad >> 15 & 1u) | bad >> 30;
                                if (i < 16) low |= two << 2 * i;
                                else high |= two << (2 * i - 32);
                                w = finite_part<T>(w);
                            }
                        }
                        // (of all: the other 64 dims of the slot may hold one)
                        *reinterpret_cast<uint2*>(map + e % kTile * S::kWords + e / kTile * 2) = make_uint2(low, high);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    bar_sync(2 + group, cleaners);
                    if (me < 4) bad_words[12 * group + 4 * ((n + 2) % 3) + me] = 0;  // read two barriers ago, used after the next one
                }
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    wait(s_full(x, half), done & 1);
                    __syncwarp();
                    tc_after();
                    if (works) {
                        float s[64];
                        ld(s_tm + 64 * half, s);
                        if (edge) {
                            const int first = slot + 64 * half;
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint32_t seen = t >= 0 ? seen_bits(a, it, t, first + 32 * i) : 0u;
                                if (no_page)
                                    seen &= (first + 32 * i < it.sees && has_page(a, it.b, first + 32 * i) ? 0xffffu : 0u) |
                                            (first + 32 * i + 16 < it.sees && has_page(a, it.b, first + 32 * i + 16) ? 0xffff0000u : 0u);
#pragma unroll 1
                                for (uint32_t bad = seen & words[2 * half + i]; bad != 0; bad &= bad - 1) {
#pragma unroll
                                    for (int w = 0; w < S::kWords; ++w) marks[256 * w] |= map[(64 * half + 32 * i + __ffs(bad) - 1) * S::kWords + w];
                                }
#pragma unroll
                                for (int j = 0; j < 32; ++j)
                                    if (!(seen >> j & 1u)) s[32 * i + j] = a.factor < 0.0f ? INFINITY : -INFINITY;
                            }
                        }
                        if (a.factor < 0.0f) {  // (a negative scale turns the scores)
#pragma unroll
                            for (int j = 0; j < 64; ++j) s[j] = -s[j];
                        }
                        float m[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) m[i] = fmaxf(s[i], s[4 + i]);
#pragma unroll
                        for (int j = 8; j < 64; j += 8)
#pragma unroll
                            for (int i = 0; i < 4; ++i) m[i] = max3(m[i], s[j + i], s[j + 4 + i]);
                        const float top = fmaxf(max3(m[0], m[1], m[2]), m[3]) * factor;
                        if (n == 0 && half == 0) {
                            ref = top;
                        } else if (__any_sync(0xffffffffu, top > ref + kSlack)) {
                            // O and the sum go over to a larger reference; rare, as it lags behind by up to kSlack
                            const bool move = top > ref + kSlack;
                            const float fade = !move ? 1.0f : ref == -INFINITY ? 0.0f : ex2(ref - top);
                            if (move) ref = top;
                            sum *= fade;
                            wait(o_done(x, 1 - half), (done - 1 + half) & 1);  // of the half before
                            __syncwarp();
                            tc_after();
#pragma unroll 1
                            for (int i = 0; i < d; i += 16) {
                                float o[16];
                                ld16(o_tm + i, o);
                                uint32_t w[16];
#pragma unroll
                                for (int j = 0; j < 16; ++j) w[j] = __float_as_uint(o[j] * fade);
                                st16(o_tm + i, w);
                            }
                        }
                        const float less = (ref == -INFINITY ? 0.0f : ref) - kLift;
                        const uint64_t by = pair(factor, factor), off = pair(-less, -less);
                        if (twice) bar_sync(4 + x, 256);
                        sum += probabilities<T>(s, by, off, s_tm + 64 * half);
                        if (twice) bar_arrive(5 - x, 256);
                        wait_st();
                    } else if (twice) {
                        bar_sync(4 + x, 256);
                        bar_arrive(5 - x, 256);
                    }
                    tc_before();
                    __syncwarp();
                    if (lane == 0) dev::mbar_arrive(p_full(x, half));
                }
            }
            unit0 += 2 * (to - from);
            if (n > 0) {
                wait(o_done(x, 1), (done - 1) & 1);
                __syncwarp();
                tc_after();
            }
            const bool whole = from == 0 && to == it.tiles;
            // the part of an item that an earlier CTA began is the CTA's part 0, of one that goes on its part 1
            float* const part = parts + (static_cast<int64_t>(blockIdx.x) * 2 + (from == 0)) * S::kPart;
            float* const there = reinterpret_cast<float*>(smem + (warp % 4) * (HDP * 128));  // [HDP / 4][32 rows][4], over the queries
            float* const stats = reinterpret_cast<float*>(smem + S::kStats);                 // [reference, sum][row]
            float total = sum, by = 1.0f, with = 0.0f, common = ref;
            auto mark = [&](float (&o)[64], int i) {  // NaN in the vector's marked dims, of 64 from i
                const uint32_t low = marks[256 * (i / 32)], high = marks[256 * (i / 32 + 1)];
                if (__any_sync(0xffffffffu, (low | high) != 0)) [[unlikely]] {
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if ((j < 32 ? low : high) >> (j % 32) & 1u) o[j] = __uint_as_float(0x7fc00000u);
                }
            };
            if (!twice) {  // the second stream's results go to the first
                bar_sync(1, 256);  // nothing reads the queries any more
                if (x == 1) {
                    stats[row] = ref, stats[kLanes + row] = sum;
                    if (works && n > 0) {
#pragma unroll 1
                        for (int i = 0; i < HDP; i += 64) {
                            float o[64];
                            ld(o_tm + i, o);
                            mark(o, i);
#pragma unroll
                            for (int j = 0; j < 64; j += 4)
                                *reinterpret_cast<float4*>(there + ((i + j) / 4 * 32 + lane) * 4) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                        }
                        tc_before();
                    }
                }
                bar_sync(1, 256);
                if (x == 0) {
                    const float ref1 = stats[row], sum1 = stats[kLanes + row];
                    common = fmaxf(ref, ref1);
                    by = sum == 0.0f ? 0.0f : ex2(ref - common);
                    with = sum1 == 0.0f ? 0.0f : ex2(ref1 - common);
                    total = by * sum + with * sum1;
                }
            }
            if (works && (twice || x == 0)) {
                const float scale = whole ? (total == 0.0f ? 0.0f : by / total) : by;
                const float scale1 = whole ? (total == 0.0f ? 0.0f : with / total) : with;
                const int64_t at = v < it.valid ? place_of(a, it.b, it.head, it.v0 + v, static_cast<int64_t>(a.heads) * d) : 0;
                const bool staged = whole && !a.out_f32 && (a.aligned & 2);
                // 16-bit results pass through shared memory, [piece of 8 dims][row], and leave it row by row
                uint4* const stage = twice ? reinterpret_cast<uint4*>(smem + x * S::kUnit + (warp % 4) * (HDP * 64)) : reinterpret_cast<uint4*>(there);
#pragma unroll 1
                for (int i = 0; i < HDP; i += 64) {
                    float o[64];
                    ld(o_tm + i, o);
                    mark(o, i);
#pragma unroll
                    for (int j = 0; j < 64; ++j) o[j] *= scale;
                    if (!twice && to - from > 1) {  // (the second stream had a tile)
#pragma unroll
                        for (int j = 0; j < 64; j += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(there + ((i + j) / 4 * 32 + lane) * 4);
                            o[j] = fmaf(f.x, scale1, o[j]), o[j + 1] = fmaf(f.y, scale1, o[j + 1]);
                            o[j + 2] = fmaf(f.z, scale1, o[j + 2]), o[j + 3] = fmaf(f.w, scale1, o[j + 3]);
                        }
                    }
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < 64; j += 2) {  // (nan_if_infinite)
                            const uint64_t y = pair(o[j], o[j + 1]);
                            unpair(fma2(y, pair(0.0f, 0.0f), y), o[j], o[j + 1]);
                        }
                    }
                    __syncwarp();
                    if (staged) {  // (over the second stream's, which are read as far as this reaches)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            stage[(i / 8 + j) * 32 + (lane ^ j)] = make_uint4(Half16<T>::pack(o[8 * j], o[8 * j + 1]), Half16<T>::pack(o[8 * j + 2], o[8 * j + 3]),
                                                                              Half16<T>::pack(o[8 * j + 4], o[8 * j + 5]), Half16<T>::pack(o[8 * j + 6], o[8 * j + 7]));
                    } else if (v < it.valid && !whole) {
#pragma unroll
                        for (int j = 0; j < 64; j += 4)
                            __stcg(reinterpret_cast<float4*>(part + ((i + j) / 4 * kVectors + v) * 4), make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]));
                    } else if (v < it.valid) {
#pragma unroll
                        for (int j = 0; j < 64; j += 4)
                            if (i + j < d) put4<T>(a, at + i + j, make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]));
                    }
                    __syncwarp();
                }
                if (staged) {
                    const int pieces = d / 8, some = 32 / pieces;
                    int r = lane / pieces, c = lane - r * pieces;
#pragma unroll 4
                    for (int i = 0; i < pieces; ++i) {
                        const int64_t to_row = __shfl_sync(0xffffffffu, at, r);
                        if (v - lane + r < it.valid)
                            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + to_row + 8 * c) = stage[c * 32 + (r ^ (c & 7))];
                        r += some, c += 32 - some * pieces;
                        if (c >= pieces) c -= pieces, ++r;
                    }
                }
                if (!whole && v < it.valid) {
                    __stcg(part + kVectors * HDP + v, common);
                    __stcg(part + kVectors * (HDP + 1) + v, total);
                }
                tc_before();
            }
            if (threadIdx.x == 0 && from == 0 && !whole) {
                const int c1 = work.last_cta(it);
                cuts[blockIdx.x] = Cut{c1 - static_cast<int>(blockIdx.x) + 1, it.b, it.head, it.v0, it.valid, {}};
            }
        } while (work.next());
        if (x == 0) bar_sync(4, 256);  // the last turn is nobody's
    } else {
        if (warp < kCopyWarp && lane == 0) {
            // A stream's products, half a tile at a time: P V, then Q K^T of its next tile's half into the same columns, in the
            // order of issue.  The other half is with the softmax warps meanwhile.
            constexpr uint32_t kType = Half16<T>::kUmma;
            constexpr uint32_t kIdescS = (1u << 4) | kType | (static_cast<uint32_t>(kTile / 2 >> 3) << 17) | (static_cast<uint32_t>(kLanes >> 4) << 24);
            // the second product's B is MN-major (bit 16)
            constexpr uint32_t kIdescO = (1u << 4) | kType | (1u << 16) | (static_cast<uint32_t>(HDP >> 3) << 17) |
                                         (static_cast<uint32_t>(kLanes >> 4) << 24);
            const int x = warp - kIssueWarp;
            const uint32_t s_tm = tmem + kLanes * x, o_tm = tmem + S::kO + HDP * x;
            int64_t unit0 = 0;
            uint32_t items = 0, done = 0;
            while (ok) {
                const int n = it.to - it.from;
                if (n > 0) {
                    const bool twice = it.valid > kLanes;
                    const int step = twice ? 1 : 2, first = twice ? 0 : x;
                    const uint32_t qd = desc_of(base + (twice ? x * S::kUnit : 0), 16);
                    auto unit_of = [&](int64_t u) { return static_cast<int>(u % S::kUnits); };
                    auto release = [&](int u) {  // (two arrivals free a unit: one of each stream, or both of the one that uses it)
                        mma_commit(empty(u));
                        if (!twice) mma_commit(empty(u));
                    };
                    auto scores = [&](int i, int half) {
                        const int64_t u = unit0 + 2 * i;
                        const int at = unit_of(u);
                        const uint32_t kd = desc_of(base + S::kRing + at * S::kUnit + half * (kTile / 2 * 128), 16);
                        // (all steps, whatever head_dim is: under a condition the later ones lost their descriptors)
#pragma unroll
                        for (int k = 0; k < HDP / 16; ++k) {
                            const uint32_t off = ((k / 4) * (kTile * 128) + (k % 4) * 32) / 16;
                            mma_ss(s_tm + 64 * half, qd + off, kd + off, kIdescS, k > 0);
                        }
                        mma_commit(s_full(x, half));
                        if (half == 1) release(at);
                    };
                    // (a stream without a tile of this item has nothing else that would keep it from missing a phase)
                    dev::mbar_arrive(q_full);
                    wait(q_full, items++ & 1);
                    tc_after();
                    if (first < n) {  // (the first keys have landed too)
                        scores(first, 0);
                        scores(first, 1);
                    }
                    for (int i = first; ok && i < n; i += step, ++done) {
                        const int at = unit_of(unit0 + 2 * i + 1);  // whose values have landed, and the next tile's keys, once P is there
#pragma unroll 1
                        for (int half = 0; half < 2; ++half) {
                            const uint32_t vd = desc_of(base + S::kRing + at * S::kUnit + half * (kTile / 2 * 128), kTile * 128);
                            wait(p_full(x, half), done & 1);
                            tc_after();
#pragma unroll
                            for (int k = 0; k < kTile / 32; ++k)
                                mma_ts(o_tm, s_tm + 64 * half + 8 * k, vd + k * 2048 / 16, kIdescO, i > first || half > 0 || k > 0);
                            mma_commit(o_done(x, half));
                            if (half == 1) release(at);
                            if (i + step < n) scores(i + step, half);
                        }
                    }
                    unit0 += 2 * n;
                }
                if (it.last) break;
                work.step();
            }
            // no product of this stream is under way past this point, also where a wait has given up
            mma_commit(finished);
            if (!wait_counted(finished, 0)) ok = false;
        } else if (warp == kLandWarp && lane == 0) {
            // Waits for keys and values in place of the issuing warps (a wait takes them 300 clocks even when the phase is
            // over: a prompt of 4093 rows 150 us, with this 141): for an item's first keys, when it joins the softmax warps in
            // telling them of the queries, and for the values of a tile and the keys of the stream's next, when it joins
            // them in telling of the tile's first P.  It sees every unit, in the ring's order at each place, and before
            // any product that frees it: no phase is mistaken for the one before or after.
            int64_t unit0 = 0;
            uint32_t items = 0, done[2] = {0, 0};
            while (ok) {
                const int n = it.to - it.from;
                if (n > 0) {
                    const bool twice = it.valid > kLanes;
                    auto landed = [&](int64_t u) { wait(full(static_cast<int>(u % S::kUnits)), (u / S::kUnits) & 1); };
                    landed(unit0);
                    if (!twice && n > 1) landed(unit0 + 2);
                    dev::mbar_arrive(q_full);
                    wait(q_full, items++ & 1);  // (one arrival a phase)
                    for (int i = 0; ok && i < n; ++i) {
                        const int next = i + (twice ? 1 : 2);
                        landed(unit0 + 2 * i + 1);
                        if (next < n) landed(unit0 + 2 * next);
                        for (int x = twice ? 0 : i & 1; x <= (twice ? 1 : i & 1); ++x) {
                            if (done[x] > 0) wait(p_full(x, 0), (done[x] - 1) & 1);  // (one arrival a phase)
                            ++done[x];
                            dev::mbar_arrive(p_full(x, 0));
                        }
                    }
                    unit0 += 2 * n;
                }
                if (it.last) break;
                work.step();
            }
        } else if (warp == kCopyWarp) {
            // A lane has a box (64 dims of the slots of a page) of the keys' or values' unit.
            const int box = min(kPagedBox, 1 << a.page_shift), boxes = kTile / box;
            const int mine = lane % boxes, block = lane / boxes % S::kBlocks;
            const bool copies = lane < boxes * S::kBlocks;
            int64_t unit = 0;
            do {
                for (int tile = it.from, to = it.to; tile < to; ++tile) {
                    const int slot = tile * kTile + mine * box;
                    int page = -1;
                    if (copies && slot < it.sees) page = a.table[static_cast<int64_t>(it.b) * a.table_stride + (slot >> a.page_shift)];
                    const bool here = page >= 0 && page < a.pages;
                    const uint32_t who = __ballot_sync(0xffffffffu, here);
                    const int first = here ? ((page * a.kv_heads + it.head) << a.page_shift) + (slot & ((1 << a.page_shift) - 1)) : 0;
#pragma unroll
                    for (int v = 0; v < 2; ++v, ++unit) {
                        const int x = static_cast<int>(unit % S::kUnits);
                        if (unit >= S::kUnits) wait(empty(x), (unit / S::kUnits - 1) & 1);
                        if (!__all_sync(0xffffffffu, ok)) break;
                        if (lane == 0) dev::mbar_expect_tx(full(x), __popc(who) * box * 128);
                        __syncwarp();
                        if (here)
                            dev::tma_load_2d(base + S::kRing + x * S::kUnit + block * (kTile * 128) + mine * box * 128, v ? &v_map : &k_map,
                                             block * 64, first, full(x));
                    }
                    if (!__all_sync(0xffffffffu, ok)) break;
                }
            } while (__all_sync(0xffffffffu, ok) && work.next());
            zero_rows(a);
            // no copy is in flight past this point, also where a wait has given up
            for (int64_t u = max(static_cast<int64_t>(0), unit - S::kUnits); u < unit; ++u)
                if (!wait_counted(full(static_cast<int>(u % S::kUnits)), (u / S::kUnits) & 1)) ok = false;
        }
        __syncwarp();
    }
    if (!ok) atomicOr(err, 1);
    tc_before();
    __syncthreads();
    if (warp == kIssueWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Items that were cut, from their parts: a thread has four dims of a vector, and the loads of
// four parts under way.
template <typename T, int HDP>
__global__ void __launch_bounds__(256) paged_merge_kernel(const __grid_constant__ PagedAttention a) {
    using S = ManyShape<HDP>;
    dev::pdl_wait();
    dev::pdl_launch_dependents();
    const Cut cut = reinterpret_cast<const Cut*>(static_cast<const char*>(a.scratch) + kPagedCounterBytes)[blockIdx.x];
    const int v = blockIdx.y * 32 + threadIdx.x % 32, quad = blockIdx.z * 8 + threadIdx.x / 32;
    if (cut.parts == 0 || v >= cut.valid || 4 * quad >= a.head_dim) return;
    const float* const parts = reinterpret_cast<const float*>(static_cast<const char*>(a.scratch) + kPagedPartsAt) +
                               static_cast<int64_t>(blockIdx.x) * 2 * S::kPart;
    float top = -INFINITY, total = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int i = 0; i < cut.parts; i += 4) {
        float ref[4], sum[4];
        float4 f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // the first is its CTA's part 1, the others are their CTAs' parts 0
            const float* const part = parts + static_cast<int64_t>(i + j == 0 ? 1 : 2 * min(i + j, cut.parts - 1)) * S::kPart;
            ref[j] = part[kVectors * HDP + v];
            sum[j] = i + j < cut.parts ? part[kVectors * (HDP + 1) + v] : 0.0f;
            f[j] = *reinterpret_cast<const float4*>(part + (quad * kVectors + v) * 4);
        }
        float now = top;
#pragma unroll
        for (int j = 0; j < 4; ++j) now = fmaxf(now, ref[j]);
        const float fade = total == 0.0f ? 0.0f : ex2(top - now);
        top = now;
        total *= fade, y.x *= fade, y.y *= fade, y.z *= fade, y.w *= fade;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float w = sum[j] == 0.0f ? 0.0f : ex2(ref[j] - top);
            total += w * sum[j];
            y.x += w * f[j].x, y.y += w * f[j].y, y.z += w * f[j].z, y.w += w * f[j].w;
        }
    }
    const float scale = total == 0.0f ? 0.0f : 1.0f / total;
    put4<T>(a, place_of(a, cut.b, cut.head, cut.v0 + v, static_cast<int64_t>(a.heads) * a.head_dim) + 4 * quad,
            make_float4(nan_if_infinite(y.x * scale), nan_if_infinite(y.y * scale), nan_if_infinite(y.z * scale), nan_if_infinite(y.w * scale)));
}

template <typename T, int HDP>
cudaError_t launch(const CUtensorMap& k_map, const CUtensorMap& v_map, const PagedAttention& a, int sm_count, int32_t* err,
                   cudaStream_t s) {
    using S = ManyShape<HDP>;
    static std::atomic<uint64_t> allowed{0};
    const auto kernel = paged_many_kernel<T, HDP>;
    cudaError_t e = allow_shared(kernel, S::kSmem, allowed);
    if (e != cudaSuccess) return e;
    const int64_t items = static_cast<int64_t>(a.batch) * a.kv_heads * ((static_cast<int64_t>(a.rows) * a.group + kVectors - 1) / kVectors);
    const int64_t most = std::max(items, items * ((a.capacity + kTile - 1) / kTile) / kLeast);
    const int grid = static_cast<int>(std::min<int64_t>(std::min(sm_count, kPagedManyCtas), most));
    e = launch_dependent(kernel, dim3(grid), dim3(kThreads), S::kSmem, s, k_map, v_map, a, err);
    // (one sequence's items are dealt or not by numbers known here; dealt ones have no parts)
    const bool dealt = a.batch == 1 && items > a.kv_heads && items >= static_cast<int64_t>(kDeal) * grid;
    if (e == cudaSuccess && !dealt) e = launch_dependent(paged_merge_kernel<T, HDP>, dim3(grid, kVectors / 32, HDP / 32), dim3(256), 0, s, a);
    return e;
}

}  // namespace

size_t paged_many_bytes(int sm_count) {
    return static_cast<size_t>(std::min(sm_count, kPagedManyCtas)) * 2 * ManyShape<128>::kPart * sizeof(float);
}

cudaError_t launch_paged_many(bool bf16, const CUtensorMap (&maps)[2], const PagedAttention& a, int sm_count, int32_t* err,
                              cudaStream_t s) {
    const bool wide = a.head_dim > 64;
    const auto run = bf16 ? wide ? launch<__nv_bfloat16, 128> : launch<__nv_bfloat16, 64>
                          : wide ? launch<__half, 128> : launch<__half, 64>;
    return run(maps[0], maps[1], a, sm_count, err, s);
}

}  // namespace kt
