// Attention over the paged latent cache: queries [tokens, heads, 512] against cached rows of 448 e4m3 values with power-of-two scales and 64
// bf16 values, or of 448 e2m1 values with such scales (the cache in 4 bits) and those 64, which are keys and values at once.
//
//   s_j = scale * q . k_j over the keys a token sees, o = sum_j e^(s_j - m) k_j / (sum_j e^(s_j - m) + e^(sink - m)), lse = m + ln sum_j e^(s_j - m)
//
// in one pass over the keys with a running maximum m and sum.  Both products run on the tensor cores with fp32 accumulators in TMEM.
//
// A tile is 64 rows of q that share a list of keys: the heads of one token (64 of them at a time), or of several neighbouring tokens of a
// request where there are fewer heads.  A CTA of 20 warps holds a tile's q (64 KiB) and streams its keys in blocks of 48, three of them in flight:
//   warps 0-3    "softmax": S from TMEM, masks, running maximum and sum, P as bf16 to shared memory; O is multiplied by a correction only where a row's
//                maximum has grown by more than a factor of 2^8 (P and the sum may exceed one by that factor; fp32 holds them).  At a tile's end: O to the
//                output, or to the workspace as a piece.  P is the one value that is held in fewer bits than its definition's: the products take operands of 16, and both
//                of one type, which the keys fix (bf16 holds them all, fp16 does not).  A weight is off by at most 2^-8 of itself, the sum of the weights stays in fp32;
//                against 64 bits `out` is off by 0.0017 to 0.0022 of its norm, where rounding it to bf16 alone makes 0.0017.
//   warps 4-15   "readers": four keys of each block a warp.  They convert the cached rows to bf16 and store them swizzled, once; the same bytes are the
//                K-major operand of S = Q K^T and the MN-major operand of O += P V.
//   warp 16      one elected lane issues the products: S of the next block before O of this one, so that they run while the softmax does.
//   warp 17      looks the next two blocks' keys up (block table or list of slots) and tells the readers where they are.
//   warps 18-19  copy q of the next tile as soon as the last S of this one is done.
// O takes 64 x 512 accumulators: 256 columns, dimensions 0-255 in lanes 0-15 of each 32 and 256-511 in lanes 16-31 (a product of 64 rows uses
// 16 lanes of each 32).
//
// Rows of work are few in decoding and of any length, so the blocks of all tiles are dealt out evenly: every CTA computes the same prefix sum
// over the tiles' numbers of blocks and takes its share, which may begin and end inside a tile.  Pieces of a tile go to a workspace as
// unnormalised sums and are joined, in a fixed order, by a second small kernel.  Where lists are short, tiles are not cut (see kLeastSplit).
//
// What bounds it.  Products of 64 rows run at half the rate: 28 cycles of a depth of 16 for the 48 columns of S (its operands come out of shared memory at
// 128 bytes a cycle), 128 for 256 columns of O, 1664 cycles a block as bare products, which a block of the largest chunk takes 2110 to 2190 of at 1.7 to 1.84 GHz: steps
// that save cycles there cost clock, at 1000 W.  A look at a barrier takes 150 to 250 cycles beside them, so softmax (1150 cycles from S to P) and readers (1700 to
// 2000 a block: look-up 170, asking 300, the stage 170, conversion 700 to 1000, handing over 150, and what the loads take) are not far behind.
// At a tile's end O goes out in 6000 to 7000 cycles of the four softmax warps, in which no product runs; the next tile's keys and first S are there before that.
// In one CTA 128 rows would need 128 KiB for q and 512 columns for O, and leave nothing for S.  A pair of CTAs with 64 rows of q each needs neither, in products
// that both take part in (cta_group::2: 64.9 cycles for the same 256 columns of 128 rows, 25.7 for 64); that form is timed as a bare product only, not built.
// e4m3 | 4 bits, one behind the other on the same GPU: 1024 tokens x 128 heads over 8192 keys 3.05 to 3.28 | 2.93 to 3.12 ms (720 | 760 TFLOP/s; 1.84 | 1.87 GHz at the power limit); 61 requests of up to
// 16384 keys, 64 heads, 120 | 110 us with 444 thousand keys in all, 146 | 134 us with 578 thousand, with 8 heads 138 | 128 us, with a window of 128 tokens and 4 first ones 13.2 | 12.8 us; one
// request of 65536 keys, 128 heads, 46.2 | 44.4 us; 61 tokens x 128 heads of up to 512 listed keys 24.2 | 23.6 us, 509 of up to 2048 377 | 370 us; a window of 128 tokens, one request, 11.1 us
// both, of which two thirds are the way in (plan, look-up, keys, q: each waits for memory that the one before names) and out.
// Other forms that were built: blocks of 64 keys in two stages, 6.9 ms; two groups of readers in turn, 4.5 (4 bits: 3.11 | 3.06, 122 us | 116); eight softmax warps, 4.1
// (this form then 3.9); two CTAs that share out keys and exchange S and P, 128 rows a product: 5.0, since each exchange takes 400 cycles one way; for the cache
// in 4 bits readers that ask for the next block before they convert this one (124 us | 116), a lane for a whole group of 32 values (3.08 | 3.12 ms, 113 us | 116, 376 | 370), S in
// two accumulators (the same), S and O from two issuing warps (3.3 | 3.1 ms), e2m1 by byte permutations alone (3.28 | 3.08), by products with f16 powers behind a look at
// the codes' range (111.6 us | 111.3, 3.15 ms | 3.17; without the look, which the format does not allow, 108.8 and 3.04), the issuer's products in a loop
// (3.8 | 3.1), O written out by the readers at the reuse of a tile's last stage (3.7 | 3.1: what it adds to their loop costs more than the 3 us a tile that it saves), a tile
// counted as three to five blocks when they are dealt out (the same).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dsv4_common.cuh"
#include "latent_attention.cuh"

namespace dsv4 {

__device__ int g_attention_error = 0;

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRows = 64, kBlockKeys = 48, kStages = 3;
constexpr int kSoftmaxWarps = 4, kReaderWarps = 12, kIssuerWarp = kSoftmaxWarps + kReaderWarps, kLookupWarp = kIssuerWarp + 1, kQueryWarps = 2;
constexpr int kThreads = 32 * (kLookupWarp + 1 + kQueryWarps), kWarpKeys = kBlockKeys / kReaderWarps;
// Registers a thread: 96 at launch (65536 / 640 threads, in steps of 8), then other shares of the same sum for the softmax and the readers.  All threads of a
// warpgroup (four warps) must execute the same setmaxnreg instruction, so roles that have one are whole warpgroups; the last warpgroup, which has three roles, keeps its 96.
constexpr int kSoftmaxRegisters = 128, kReaderRegisters = 80, kLaunchRegisters = 96;
static_assert(kThreads == 640 && kWarpKeys == 4, "");
static_assert(kSoftmaxWarps * kSoftmaxRegisters + kReaderWarps * kReaderRegisters + (20 - kSoftmaxWarps - kReaderWarps) * kLaunchRegisters <= 20 * kLaunchRegisters, "");
static_assert(kSoftmaxWarps % 4 == 0 && kReaderWarps % 4 == 0, "whole warpgroups");
constexpr uint64_t kAllKeys = (1ull << kBlockKeys) - 1;
constexpr float kMostGrowth = 8.0f;  // log2 of the factor that a row's maximum may have grown by before O is corrected (with 0: 61 requests 209 us, not 155)
constexpr int kLookChunk = 6;  // of S's eight chunks, the one in front of which P is looked for (4, 6, 7: 3172, 3167, 3174 us)
constexpr int kMaxCtas = 148;        // a B200's SMs: one CTA on each (its shared memory allows no second)
// Splitting.  A piece costs 128 KiB of fp32 sums out and in, and the kernel that joins them 6 to 10 us, so no tile shorter than kLeastSplit blocks is cut
// (with 8: 61 tokens x 128 heads of up to 512 listed keys 38 us, with 16: 24; a chunk with a window of 512: 515 | 462; one request of 700 keys: 24.7 | 26.6);
// no piece is shorter than kLeastPiece (61 requests of up to 16384 keys: with 2 154.5 us, with 4 152.6); and a CTA has at least kLeastShare blocks (with 3, 4, 5
// and 6, one request of 700 keys: 26.3, 27.4, 25.4, 27.7 us).
// Where every tile can have a CTA and none is longer than kMostWhole blocks, they stay whole if that costs the longest no more than kSplitCost blocks over an even
// share (61 x 128 heads of up to 1000 keys: 36 us, cut 49; 8 x 128 heads of up to 700: 26.8, cut 26.5).  The CTA of each is then its number, which saves the
// plan (one request, a window of 128: 12.1 us, with a plan 13.8).  Beyond kMostWhole a batch of one long and many short lists would lose too much.
constexpr int kLeastPiece = 4, kLeastShare = 5, kLeastSplit = 16, kSplitCost = 12, kMostWhole = 24;

// ---- shared memory -----------------------------------------------------------------------------------------------------------

constexpr int kQueryChunk = kRows * 128, kKeyChunk = kBlockKeys * 128;  // rows of 64 dimensions: 8-row, 128-byte swizzle atoms
constexpr int kQueryBytes = 8 * kQueryChunk, kKeyBytes = 8 * kKeyChunk;   // 64 KiB and 48 KiB
constexpr int kOffsetKeys = kQueryBytes, kOffsetP = kOffsetKeys + kStages * kKeyBytes, kOffsetRest = kOffsetP + 2 * kQueryChunk;

struct Cut {
    int request, token, group, block;
};
struct Rest {
    uint64_t kv_full[kStages], kv_empty[kStages], s_full[2], p_full[2], pv_done[2], look_full[2], look_empty[2], q_full, q_empty, o_empty, drained;
    uint64_t sums[kThreads / 32];
    uint64_t valid[kStages];                        // a bit per key of a block: it exists,
    alignas(4) uint8_t bad[kStages][kReaderWarps];  // it has a value that is not finite: four keys a reader warp (mixed blocks only)
    // What the look-up warp tells the readers of the next two blocks: where the values and the scale codes of every key are, which exist (bit 63:
    // there is no such block), and whether the block is mixed.
    alignas(16) ulonglong2 keys[2][kBlockKeys];
    uint64_t exist[2];
    uint32_t mixed[2];
    Cut from, to;
    uint32_t tmem;
    int abort;
};
constexpr int kSharedBytes = kOffsetRest + static_cast<int>(sizeof(Rest));
static_assert(kSharedBytes <= 232448, "227 KiB a CTA");
constexpr int kScratchInts = kOffsetRest / 4;  // all that is not in use while the plan is made

// ---- PTX ----------------------------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(bar)) : "memory");
}
constexpr uint32_t kTryNs = 2000;  // how long the hardware may suspend the thread in one try
__device__ __forceinline__ bool barrier_try(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(shared_address(bar)), "r"(parity), "r"(kTryNs)
                 : "memory");
    return done != 0;
}
// Whether the phase has completed, at once.
__device__ __forceinline__ uint32_t barrier_test(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(shared_address(bar)), "r"(parity)
                 : "memory");
    return done;
}
// What bounds a wait: a number of tries behind the first (launch parameter), each of which the hardware suspends for up to two microseconds, and the
// word by which a role that has given up tells the CTA's others to leave.
struct Limit {
    volatile int* abort;
    uint32_t retries;
};
// False, and the others told, where the phase does not complete within the limit.  (The default allows some seconds; a phase takes a few microseconds.)
// The limit is looked at behind a try that failed: ahead of the first one, sparse 61 tokens 24.5 us, 61 requests 157, not 24.1 and 155.5.
__device__ __forceinline__ bool barrier_wait(uint64_t* bar, uint32_t parity, const Limit& limit) {
    for (uint32_t i = 0;; ++i) {
        if (barrier_try(bar, parity)) return true;
        if (*limit.abort) return false;
        if (i >= limit.retries) break;
    }
    *limit.abort = 1;
    atomicOr(&g_attention_error, 1);
    return false;
}
// The same by a whole warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const Limit& limit) {
    return __all_sync(0xffffffffu, barrier_wait(bar, parity, limit));
}
// Between a thread's ordinary writes of shared memory and the products that read them.  It waits for the thread's loads that are under way, too.
__device__ __forceinline__ void fence_to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_tmem_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void commit_to(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(bar)) : "memory");
}
__device__ __forceinline__ void multiply(uint32_t d, uint64_t a, uint64_t b, uint32_t kind, bool accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(kind), "r"(static_cast<uint32_t>(accumulate))
                 : "memory");
}
// One lane of a converged warp.  A branch on it, unlike one on a lane's number, lets the compiler keep descriptors in uniform registers: a
// product of 64 x 64 x 16 is issued every 33 cycles (its rate) instead of every 45.
__device__ __forceinline__ bool elected() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
#define DSV4_R8(v, i) "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]), "=f"(v[i + 4]), "=f"(v[i + 5]), "=f"(v[i + 6]), "=f"(v[i + 7])
#define DSV4_W8(v, i) "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]), "f"(v[i + 6]), "f"(v[i + 7])
#define DSV4_LIST32                                                                                                                       \
    "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}"
// 16 lanes x 48 columns: lane l of the warp gets, of columns 8j + 2(l % 4) + {0, 1}, row l / 4 in v[4j], v[4j + 1] and row l / 4 + 8 in the
// next two.
__device__ __forceinline__ void load_scores(float (&v)[24], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : DSV4_R8(v, 0), DSV4_R8(v, 8)
                 : "r"(at));
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];" : DSV4_R8(v, 16) : "r"(at + 32));
}
// 32 lanes x 32 columns, one lane a thread.
__device__ __forceinline__ void load_columns(float (&v)[32], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 " DSV4_LIST32 ", [%32];"
                 : DSV4_R8(v, 0), DSV4_R8(v, 8), DSV4_R8(v, 16), DSV4_R8(v, 24)
                 : "r"(at));
}
// Behind the loads of v: names it, so that nothing that uses it moves ahead of the wait.
#define DSV4_U8(v, i) "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7])
__device__ __forceinline__ void wait_tmem_loads(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : DSV4_U8(v, 0), DSV4_U8(v, 8), DSV4_U8(v, 16), DSV4_U8(v, 24)::"memory");
}
__device__ __forceinline__ void wait_tmem_loads(float (&v)[24]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : DSV4_U8(v, 0), DSV4_U8(v, 8), DSV4_U8(v, 16)::"memory");
}
__device__ __forceinline__ void store_columns(const float (&v)[32], uint32_t at) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], " DSV4_LIST32 ";" ::DSV4_W8(v, 0), DSV4_W8(v, 8), DSV4_W8(v, 16), DSV4_W8(v, 24),
                 "r"(at)
                 : "memory");
}
__device__ __forceinline__ void store_shared16(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void store_shared4(uint32_t at, uint32_t v) { asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// max(a, b, c), two products and sums at once: one instruction each
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 y;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(y.x), "=f"(y.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return y;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 y;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(y.x), "=f"(y.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return y;
}

// Shared-memory operand with 128-byte swizzle: atoms of 8 rows x 128 bytes, the next 8 rows 1024 bytes on.  `leading`: bytes between chunks of
// 64 dimensions, used where the dimensions are the operand's outer direction.
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t leading) {
    return static_cast<uint64_t>((address & 0x3ffffu) >> 4) | (static_cast<uint64_t>(leading >> 4) << 16) | (static_cast<uint64_t>(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// bf16 x bf16 -> fp32, 64 rows, n columns; `transposed`: the second operand's columns are contiguous.
constexpr uint32_t kind_of(uint32_t n, bool transposed) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (transposed ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((kRows >> 4) << 24);
}

constexpr uint32_t kKindS = kind_of(kBlockKeys, false), kKindO = kind_of(256, true);

// ---- tiles and their order ------------------------------------------------------------------------------------------------------

// The lists of starts and lengths, in global memory or, while the plan is made, copied to shared memory.
struct Lists {
    const int32_t *starts, *lens;
};
struct Tiles {
    LatentAttention a;
    Lists lists;
    int32_t tokens_per_tile, head_groups;
    int32_t one_each;  // every CTA has the whole tile of its number, if there is one
    float* sums;      // workspace: [2 * kMaxCtas][64][512] unnormalised outputs,
    float2* rows;     // [2 * kMaxCtas][64] their maximum and sum,
    int4* pieces;     // [2 * kMaxCtas] what they belong to: token, first head, rows, and 0: nothing, 1: more follow, 2: the last
};

// The keys of a tile as one list: `first` first tokens, then the positions from `low` on.
struct Tile {
    int token, count, head, rows, position, first, low, keys, blocks;
    // Whether some rows of the tile see a key of the block that others do not.
    __device__ __forceinline__ bool mixed(const Tiles& p, int block) const {
        if (count == 1) return false;
        const int k0 = block * kBlockKeys, k1 = min(k0 + kBlockKeys, keys) - 1;
        const int oldest = k0 < first ? k0 : k0 - first + low, newest = k1 < first ? k1 : k1 - first + low;
        return newest > position || (p.a.window > 0 && (k0 < first || oldest <= position + count - 1 - p.a.window));
    }
};

__device__ __forceinline__ Tile tile_at(const Tiles& p, const Lists& lists, int request, int token, int group) {
    Tile t;
    t.token = token, t.head = group * kRows;
    t.position = t.first = t.low = 0;
    if (p.a.indices) {
        t.count = 1;
        t.keys = min(max(lists.lens[token], 0), p.a.topk);
    } else {
        const int end = lists.starts[request + 1];  // (it may lie behind the last row of q: positions count from it all the same)
        t.count = min(p.tokens_per_tile, min(end, p.a.num_tokens) - token);
        t.position = max(lists.lens[request], 0) - end + token;
        t.low = p.a.window > 0 && t.position >= p.a.window ? t.position - p.a.window + 1 : 0;
        t.first = min(min(t.low, p.a.first), p.a.capacity);
        t.keys = max(0, min(t.position + t.count, p.a.capacity) - t.low) + t.first;
    }
    t.rows = p.head_groups > 1 ? min(kRows, p.a.num_heads - t.head) : t.count * p.a.num_heads;
    t.blocks = static_cast<int>((static_cast<uint32_t>(t.keys) + kBlockKeys - 1) / kBlockKeys);
    return t;
}

// Request of the first token at or behind `token` that belongs to one (num_reqs if none does), and that token.
__device__ __forceinline__ int request_of(const Tiles& p, const Lists& lists, int& token) {
    if (p.a.indices) return 0;
    token = max(token, lists.starts[0]);
    int low = 0, high = p.a.num_reqs;  // the first request that ends behind the token
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (lists.starts[mid + 1] > token) high = mid;
        else low = mid + 1;
    }
    return low;
}

// A CTA's share: pieces of tiles, in order.
struct Walk {
    Cut at;
    const Cut* end_of_share;  // in shared memory
    Tile tile;
    int begin, end;  // blocks of the tile
    __device__ __forceinline__ void step(const Tiles& p) {
        if (++at.group == p.head_groups) {
            at.group = 0;
            at.token += tile.count;
            if (!p.a.indices)
                while (at.request < p.a.num_reqs && __ldg(p.lists.starts + at.request + 1) <= at.token) ++at.request;
            if (at.request >= p.a.num_reqs && !p.a.indices) at.token = p.a.num_tokens;
        }
        at.block = 0;
    }
    // Makes `tile`, `begin` and `end` those of the piece at `at`, or of the first one behind it that is none of nothing; false at the end.
    __device__ __forceinline__ bool settle(const Tiles& p) {
        for (;;) {
            const volatile Cut& to = *end_of_share;
            if (at.token >= p.a.num_tokens || at.token > to.token || (at.token == to.token && at.group > to.group)) return false;
            const bool last = at.token == to.token && at.group == to.group;
            if (last && to.block == 0) return false;
            tile = tile_at(p, p.lists, at.request, at.token, at.group);
            begin = at.block, end = last ? min(to.block, tile.blocks) : tile.blocks;
            if (begin < end || tile.blocks == 0) return true;
            step(p);
        }
    }
    __device__ __forceinline__ bool whole() const { return begin == 0 && end == tile.blocks; }
};

// Every CTA's share has the same number of blocks, a tile counting one more for its own cost.  All threads take part; thread-uniform results in
// rest.from and rest.to.
__device__ __forceinline__ void make_plan(const Tiles& p, Rest& rest, int32_t* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // The starts and lengths of all requests (lengths of all tokens) are read at once, where they fit, instead of in a chain of dependent loads.
    Lists lists = p.lists;
    const int starts = p.a.indices ? 0 : p.a.num_reqs + 1, lens = p.a.indices ? p.a.num_tokens : p.a.num_reqs;
    if (starts + lens <= kScratchInts) {
        for (int i = tid; i < starts; i += kThreads) scratch[i] = __ldg(p.lists.starts + i);
        for (int i = tid; i < lens; i += kThreads) scratch[starts + i] = __ldg(p.lists.lens + i);
        lists.starts = scratch, lists.lens = scratch + starts;
        __syncthreads();
    }
    const int each = (p.a.num_tokens + kThreads - 1) / kThreads;
    const int begin = min(tid * each, p.a.num_tokens), end = min(begin + each, p.a.num_tokens);
    // f(request, token, blocks) for the tiles' first tokens in [begin, end)
    const auto for_tiles = [&](auto&& f) {
        int token = begin, request = begin < end ? request_of(p, lists, token) : 0;
        while (token < end) {
            if (!p.a.indices) {
                while (request < p.a.num_reqs && lists.starts[request + 1] <= token) ++request;
                if (request >= p.a.num_reqs) break;
                const int start = lists.starts[request];
                const int behind = (token - start) % p.tokens_per_tile;
                if (behind != 0) {
                    token += p.tokens_per_tile - behind;
                    token = min(token, lists.starts[request + 1]);
                    continue;
                }
            }
            const Tile t = tile_at(p, lists, request, token, 0);
            if (f(request, token, t.blocks)) break;
            token += t.count;
        }
    };
    if (tid == 0) rest.from = rest.to = Cut{p.a.num_reqs, p.a.num_tokens, 0, 0};
    if (p.one_each) {
        __syncthreads();
        if (tid == 0) {
            const int group = blockIdx.x % p.head_groups, mine = blockIdx.x / p.head_groups;
            int token = mine;
            const int request = mine < p.a.num_tokens ? request_of(p, lists, token) : p.a.num_reqs;
            // (a token in front of the first request's, or behind the last one's, has none; nor has one in the middle of a tile)
            if (mine < p.a.num_tokens && token == mine && (p.a.indices || (request < p.a.num_reqs && (token - lists.starts[request]) % p.tokens_per_tile == 0))) {
                rest.from = Cut{request, token, group, 0};
                rest.to = Cut{request, token, group + 1, 0};
            }
        }
        __syncthreads();
        return;
    }
    uint64_t mine = 0;
    for_tiles([&](int, int, int blocks) {
        mine += static_cast<uint64_t>(blocks + 1) * p.head_groups;
        return false;
    });
    uint64_t up_to = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint64_t other = __shfl_up_sync(0xffffffffu, up_to, d);
        if (lane >= d) up_to += other;
    }
    if (lane == 31) rest.sums[warp] = up_to;
    __syncthreads();
    uint64_t total = 0, before = up_to - mine;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += rest.sums[w];
        total += rest.sums[w];
    }
    const uint64_t ctas = min(static_cast<uint64_t>(gridDim.x), max(total / kLeastShare, static_cast<uint64_t>(1)));
    for (int side = 0; side < 2; ++side) {
        const uint64_t cta = blockIdx.x + side;
        if (cta >= ctas) continue;
        const uint64_t cut = total * cta / ctas;
        if (cut < before || cut >= before + mine) continue;
        uint64_t at = before;
        for_tiles([&](int request, int token, int blocks) {
            const uint64_t next = at + static_cast<uint64_t>(blocks + 1) * p.head_groups;
            if (cut >= next) {
                at = next;
                return false;
            }
            const uint64_t behind = cut - at;  // (below 2^32 but for tiles of 2^25 blocks in hundreds of groups)
            const uint32_t each = blocks + 1, whole = p.head_groups == 1 ? 0 : behind >> 32 ? static_cast<uint32_t>(behind / each) : static_cast<uint32_t>(behind) / each;
            const int group = static_cast<int>(whole), offset = static_cast<int>(behind - static_cast<uint64_t>(whole) * each);
            int block = min(offset, blocks);
            if (blocks < kLeastSplit) block = 2 * offset <= blocks ? 0 : blocks;
            else if (block < kLeastPiece) block = 0;
            else if (blocks - block < kLeastPiece) block = blocks;
            (side == 0 ? rest.from : rest.to) = Cut{request, token, group, block};
            return true;
        });
    }
    __syncthreads();
}

// ---- the kernel -------------------------------------------------------------------------------------------------------------------

// Two e4m3 bytes of `word` (the low ones, or the high ones) times a power of two, given as a pair of equal bf16: the values are exact in bf16,
// and their product is rounded once.
template <int HIGH>
__device__ __forceinline__ uint32_t two_values(uint32_t word, uint32_t scale) {
    uint32_t halves, out;
    const auto pair = static_cast<uint16_t>(HIGH ? word >> 16 : word);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(pair));
    float lo, hi;
    asm("{.reg .f16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(lo), "=f"(hi) : "r"(halves));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(out) : "r"(pack_bf16x2(lo, hi)), "r"(scale));
    return out;
}

// 2^(code - 127) as a pair of bf16; 0: subnormal, 255: infinity.
// `codes` has the code twice, one in each half.
__device__ __forceinline__ uint32_t power_of_codes(uint32_t codes) { return __vmaxu2(codes << 7, 0x400040u); }

// The same, but 255 is NaN; the code twice in the low half.
__device__ __forceinline__ uint32_t power_of_mx_codes(uint32_t codes) {
    uint32_t v;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, l;\n\t}" : "=r"(v) : "r"(codes));
    return v;
}

// Two fp32 values that bf16 holds, as a pair: a permutation of bytes, where the conversion shares a unit with the one to f16 in front of it (509 listed tokens 368 | 374 us,
// 61 23.1 | 23.5, the others 0.3 to 0.7 % less; beside the conversions of e4m3 it costs 0 to 2 %).
__device__ __forceinline__ uint32_t upper_halves(float lo, float hi) { return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x7632); }

// Eight e2m1 values (the first in the low bits) times a power of two.
__device__ __forceinline__ uint4 eight_values(uint32_t word, uint32_t scale) {
    uint32_t h[4], v[4];
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(word));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        asm("{.reg .f16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h;}" : "=f"(lo), "=f"(hi) : "r"(h[i]));
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(v[i]) : "r"(upper_halves(lo, hi)), "r"(scale));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Whether one of a bf16 pair is infinite or NaN.
__device__ __forceinline__ bool not_finite(uint32_t pair) { return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ bool not_finite(const uint4& v) { return not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w); }

// Twelve bytes of four bits each as one number.
__device__ __forceinline__ uint64_t key_bits(const uint32_t* v) {
    const auto four = [](uint32_t x) {
        x = (x | (x >> 4)) & 0x00ff00ffu;
        return (x | (x >> 8)) & 0xffffu;
    };
    return static_cast<uint64_t>(four(v[0]) | (four(v[1]) << 16)) | (static_cast<uint64_t>(four(v[2])) << 32);
}

template <int COUNT, bool MORE>
__device__ __forceinline__ void set_registers() {
    if (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(COUNT));
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(COUNT));
}

// MX: the cache in 4 bits.
template <bool MX>
__global__ void __launch_bounds__(kThreads, 1) latent_attention_kernel(const Launched<Tiles> p) {
    constexpr int kDataBytes = MX ? kMxTokenDataBytes : kTokenDataBytes, kCodeBytes = MX ? kMxScaleBytes : kScaleBytes;
    extern __shared__ __align__(1024) uint8_t shared[];
    Rest& rest = *reinterpret_cast<Rest*>(shared + kOffsetRest);
    const uint32_t base = shared_address(shared);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) barrier_init(&rest.kv_full[i], kReaderWarps), barrier_init(&rest.kv_empty[i], 1);
        for (int i = 0; i < 2; ++i) barrier_init(&rest.s_full[i], 1), barrier_init(&rest.p_full[i], kSoftmaxWarps), barrier_init(&rest.pv_done[i], 1);
        for (int i = 0; i < 2; ++i) barrier_init(&rest.look_full[i], 1), barrier_init(&rest.look_empty[i], kReaderWarps);
        barrier_init(&rest.q_full, kQueryWarps), barrier_init(&rest.q_empty, 1), barrier_init(&rest.o_empty, kSoftmaxWarps), barrier_init(&rest.drained, 1);
        rest.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_to_async();
    }
    if (warp == kIssuerWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_address(&rest.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    begin_dependent_kernel();
    make_plan(p, rest, reinterpret_cast<int32_t*>(shared));
    fence_tmem_before();
    __syncthreads();
    fence_tmem_after();
    const uint32_t tmem = rest.tmem, tmem_scores = tmem + 256;
    const Limit limit{&rest.abort, p.a.wait_retries};
    Walk w;
    w.at = rest.from, w.end_of_share = &rest.to;

    if (warp < kSoftmaxWarps) {
        // ------------------------------------------------------------------------------------------------ softmax, outputs
        set_registers<kSoftmaxRegisters, true>();
        const float c = p.a.scale * kLog2e;
        const int row_a = 16 * warp + (lane >> 2), quad = 2 * (lane & 3);
        const uint32_t lanes = static_cast<uint32_t>(32 * warp) << 16;
        int it = 0, stage = 0;  // blocks so far, and that number modulo kStages
        uint32_t stage_phase = 0;
        bool ok = true;
        const int slot_of_head = 2 * blockIdx.x + 1, slot_of_rest = 2 * blockIdx.x;
        if (threadIdx.x < 2 && p.pieces) p.pieces[2 * blockIdx.x + threadIdx.x] = make_int4(0, 0, 0, 0);
        __syncwarp();
        for (; ok && w.settle(p); w.step(p)) {
            const Tile& t = w.tile;
            float m[2] = {-INFINITY, -INFINITY};
            float2 l[2] = {};  // (sums of even and of odd columns)
            // positions of this thread's two rows
            int position[2] = {t.position, t.position};
            if (t.count > 1) position[0] += row_a / p.a.num_heads, position[1] += (row_a + 8) / p.a.num_heads;
            for (int block = w.begin; block < w.end; ++block, ++it) {
                const int buffer = it & 1;
                const uint32_t parity = (it >> 1) & 1;
                if (!warp_wait(&rest.s_full[buffer], parity, limit) || !warp_wait(&rest.kv_full[stage], stage_phase, limit)) {
                    ok = false;
                    break;
                }
                fence_tmem_after();
                float s[24];
                load_scores(s, tmem_scores + 64 * buffer + lanes);
                const uint64_t valid = rest.valid[stage];
                const bool mixed = t.mixed(p, block);
                const int k0 = block * kBlockKeys;
                wait_tmem_loads(s);
                if (mixed) {
                    const uint64_t bad = key_bits(reinterpret_cast<const uint32_t*>(rest.bad[stage]));
#pragma unroll
                    for (int i = 0; i < 24; ++i) {
                        const int k = 8 * (i >> 2) + quad + (i & 1);
                        const int at = k0 + k, where = at < t.first ? at : at - t.first + t.low;
                        const int mine = position[(i >> 1) & 1];
                        const bool seen = ((valid >> k) & 1) != 0 && where <= mine && (p.a.window <= 0 || mine - where < p.a.window || where < p.a.first);
                        s[i] = !seen ? -INFINITY : ((bad >> k) & 1) != 0 ? NAN : s[i];
                    }
                } else if (valid != kAllKeys) {
#pragma unroll
                    for (int i = 0; i < 24; ++i)
                        if (((valid >> (8 * (i >> 2) + quad + (i & 1))) & 1) == 0) s[i] = -INFINITY;
                }
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 24; i += 2) top[(i >> 1) & 1] = max3(top[(i >> 1) & 1], s[i], s[i + 1]);
                // The common case is that no row's maximum has grown by so much that it matters: every lane sees that of its own columns.
                bool grown = false;
#pragma unroll
                for (int r = 0; r < 2; ++r) grown |= m[r] == -INFINITY ? top[r] != -INFINITY : (top[r] - m[r]) * c > kMostGrowth;
                if (__any_sync(0xffffffffu, grown)) {
                    float factor[2] = {1.0f, 1.0f};
                    bool correct = false;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                        if (m[r] == -INFINITY) {
                            m[r] = top[r];  // (O is zero so far)
                        } else if (top[r] > m[r]) {
                            factor[r] = exp2_approx((m[r] - top[r]) * c);
                            l[r].x *= factor[r], l[r].y *= factor[r];
                            m[r] = top[r];
                            correct = true;
                        }
                    }
                    if (__any_sync(0xffffffffu, correct)) {
                        // O has been written up to the block before this one
                        if (!warp_wait(&rest.pv_done[buffer ^ 1], ((it - 1) >> 1) & 1, limit)) {
                            ok = false;
                            break;
                        }
                        fence_tmem_after();
                        const int from = (lane & 7) << 2;
                        const float fa = __shfl_sync(0xffffffffu, factor[0], from), fb = __shfl_sync(0xffffffffu, factor[1], from);
                        const float f = (lane & 8) ? fb : fa;
#pragma unroll 1
                        for (int at = 0; at < 256; at += 32) {
                            float o[32];
                            load_columns(o, tmem + at + lanes);
                            wait_tmem_loads(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] *= f;
                            store_columns(o, tmem + at + lanes);
                        }
                        wait_tmem_stores();
                    }
                }
                const float mc[2] = {m[0] == -INFINITY ? 0.0f : m[0] * c, m[1] == -INFINITY ? 0.0f : m[1] * c};
#pragma unroll
                for (int i = 0; i < 24; i += 2) {
                    const int r = (i >> 1) & 1;
                    const float2 x = fma2(make_float2(s[i], s[i + 1]), make_float2(c, c), make_float2(-mc[r], -mc[r]));
                    s[i] = exp2_approx(x.x), s[i + 1] = exp2_approx(x.y);
                    l[r] = add2(l[r], make_float2(s[i], s[i + 1]));
                }
                // P of two blocks ago has been read
                if (it >= 2 && !warp_wait(&rest.pv_done[buffer], ((it >> 1) - 1) & 1, limit)) {
                    ok = false;
                    break;
                }
                const uint32_t to = base + kOffsetP + buffer * kQueryChunk + row_a * 128 + 2 * quad;
#pragma unroll
                for (int j = 0; j < kBlockKeys / 8; ++j) {
                    const uint32_t unit = (j ^ (row_a & 7)) << 4;  // (row_a + 8 has the same low bits)
                    store_shared4(to + unit, pack_bf16x2(s[4 * j], s[4 * j + 1]));
                    store_shared4(to + 8 * 128 + unit, pack_bf16x2(s[4 * j + 2], s[4 * j + 3]));
                }
                fence_to_async();
                fence_tmem_before();
                __syncwarp();
                if (lane == 0) barrier_arrive(&rest.p_full[buffer]);
                if (++stage == kStages) stage = 0, stage_phase ^= 1;
            }
            if (!ok) break;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                l[r].x += l[r].y;
                l[r].x += __shfl_xor_sync(0xffffffffu, l[r].x, 1);
                l[r].x += __shfl_xor_sync(0xffffffffu, l[r].x, 2);
            }
            // From here on a lane's row is the one it has in TMEM: 16 * warp + lane % 16, dimensions 256 * (lane / 16) on.
            const int from = (lane & 7) << 2, row = 16 * warp + (lane & 15);
            const float ma = __shfl_sync(0xffffffffu, m[0], from), mb = __shfl_sync(0xffffffffu, m[1], from);
            const float la = __shfl_sync(0xffffffffu, l[0].x, from), lb = __shfl_sync(0xffffffffu, l[1].x, from);
            const float row_m = (lane & 8) ? mb : ma, row_l = (lane & 8) ? lb : la;
            const auto out_of = [&](int of) {
                const int token = t.token + (t.count > 1 ? of / p.a.num_heads : 0), head = t.count > 1 ? of % p.a.num_heads : t.head + of;
                return p.a.out + token * p.a.out_stride_token + head * p.a.out_stride_head;
            };
            float inverse = 0.0f;
            const bool some = row_l != 0.0f, whole = w.whole();
            const int slot = w.begin == 0 ? slot_of_head : slot_of_rest;
            if (!whole) {
                if (lane < 16) p.rows[slot * kRows + row] = make_float2(row_m, row_l);
                if (threadIdx.x == 0) p.pieces[slot] = make_int4(t.token, t.head, t.rows, w.end == t.blocks ? 2 : 1);
            } else if (row < t.rows) {
                const int token = t.token + (t.count > 1 ? row / p.a.num_heads : 0), head = t.count > 1 ? row % p.a.num_heads : t.head + row;
                float total = row_l;
                if (p.a.sink && some) total += exp2_approx(fmaf(__ldg(p.a.sink + head), kLog2e, -row_m * c));
                inverse = some ? 1.0f / total : 0.0f;
                if (lane < 16 && p.a.lse)
                    p.a.lse[token * p.a.lse_stride_token + head * p.a.lse_stride_head] = some ? (row_m * c + log2f(row_l)) * kLn2 : -INFINITY;
            }
            if (w.begin == w.end) {
                if (row < t.rows) {
                    uint8_t* out = out_of(row) + 512 * (lane >> 4);
#pragma unroll 1
                    for (int i = 0; i < 512; i += 16) *reinterpret_cast<uint4*>(out + i) = make_uint4(0u, 0u, 0u, 0u);
                }
                continue;
            }
            if (!warp_wait(&rest.pv_done[(it - 1) & 1], ((it - 1) >> 1) & 1, limit)) {
                ok = false;
                break;
            }
            fence_tmem_after();
            // 128 bytes of every row at a time, of both halves of its dimensions, go through this warp's rows of the two P buffers, which have been read:
            // a store then writes four rows' 128 bytes, where a lane's own would touch 32 lines each.
            const uint32_t stage_at = base + kOffsetP + 16 * warp * 128;
            const uint32_t put = stage_at + (lane >> 4) * kQueryChunk + (lane & 15) * 128, get = stage_at + (lane >> 3) * 128;
            const int unit = lane & 7;
            uint8_t* to[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int of = 16 * warp + 4 * i + (lane >> 3);
                to[i] = of >= t.rows ? nullptr : whole ? out_of(of) + 16 * unit : reinterpret_cast<uint8_t*>(p.sums + (static_cast<int64_t>(slot) * kRows + of) * kHeadDim) + 16 * unit;
            }
            const int half_bytes = whole ? 512 : 1024;
            const auto pass_on = [&] {
                __syncwarp();
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w)
                                 : "r"(get + (i >> 2) * kQueryChunk + 4 * (i & 3) * 128 + ((unit ^ ((4 * i + (lane >> 3)) & 7)) << 4))
                                 : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (to[i]) {
                        *reinterpret_cast<uint4*>(to[i]) = v[i];
                        *reinterpret_cast<uint4*>(to[i] + half_bytes) = v[i + 4];
                        to[i] += 128;
                    }
                __syncwarp();
            };
            if (whole) {
                const uint32_t keep = some ? 0xffffffffu : 0u;
#pragma unroll 1
                for (int at = 0; at < 256; at += 64) {
                    float o[2][32];
                    load_columns(o[0], tmem + at + lanes);
                    load_columns(o[1], tmem + at + 32 + lanes);
                    wait_tmem_loads(o[0]), wait_tmem_loads(o[1]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float* from = o[i >> 2] + 8 * (i & 3);
                        uint32_t v[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = pack_bf16x2(from[2 * k] * inverse, from[2 * k + 1] * inverse) & keep;
                        store_shared16(put + ((i ^ (lane & 7)) << 4), make_uint4(v[0], v[1], v[2], v[3]));
                    }
                    pass_on();
                }
            } else {
#pragma unroll 1
                for (int at = 0; at < 256; at += 32) {
                    float o[32];
                    load_columns(o, tmem + at + lanes);
                    wait_tmem_loads(o);
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        store_shared16(put + ((i ^ (lane & 7)) << 4), make_uint4(__float_as_uint(o[4 * i]), __float_as_uint(o[4 * i + 1]), __float_as_uint(o[4 * i + 2]), __float_as_uint(o[4 * i + 3])));
                    pass_on();
                }
            }
            fence_tmem_before();
            __syncwarp();
            if (lane == 0) barrier_arrive(&rest.o_empty);
        }
    } else if (warp < kIssuerWarp) {
        // ------------------------------------------------------------------------------------------------ readers
        set_registers<kReaderRegisters, false>();
        // A warp has four keys of each block.  It asks for its values of the next block when it has handed over this one's, not before: the fence
        // and the arrival wait for a warp's loads that are under way.
        const int reader = warp - kSoftmaxWarps, sub = lane >> 1, odd = lane & 1;
        // Keys 4 * reader + 2 i + odd of a block; of each, dimensions 16 sub .. of the first half, the same of the second where they are e4m3
        // (sub 0-11), and four rotary ones.  Two neighbouring keys and four subs, which are what eight lanes store at once, hit all eight 16-byte
        // columns of the swizzle.
        const int key_a = kWarpKeys * reader + odd;
        const uint32_t store_row = base + kOffsetKeys + key_a * 128, unit = 2 * (sub & 3);
        const bool coded = sub < 12;
        const int rotary_sub = sub ^ (8 * odd);  // (the two keys' halves, so that their stores use different banks)
        // of a byte of a code word and of zeros: the byte in both halves (4 bits: in both bytes of the low half)
        const uint32_t code_select = MX ? 0x4400u + 0x11u * ((sub >> 1) & 3) : 0x4040u + 0x0101u * (sub >> 2);
        // 16 cached values to two 16-byte columns
        using Values = std::conditional_t<MX, uint2, uint4>;
        const auto convert = [&](const Values& v, uint32_t code_word, uint4& a, uint4& b) {
            const uint32_t codes = __byte_perm(code_word, 0u, code_select);
            if constexpr (MX) {
                const uint32_t scale = power_of_mx_codes(codes);
                a = eight_values(v.x, scale), b = eight_values(v.y, scale);
            } else {
                const uint32_t scale = power_of_codes(codes);
                a = make_uint4(two_values<0>(v.x, scale), two_values<1>(v.x, scale), two_values<0>(v.y, scale), two_values<1>(v.y, scale));
                b = make_uint4(two_values<0>(v.z, scale), two_values<1>(v.z, scale), two_values<0>(v.w, scale), two_values<1>(v.w, scale));
            }
        };
        uint32_t to[2][2], to_rotary[2];  // where this lane's values of the two keys go: 16-byte columns of the first half's chunk, and the rotary ones
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t twist = (key_a + 2 * i) & 7, row = store_row + 2 * i * 128;
            to[i][0] = row + (sub >> 2) * kKeyChunk + ((unit ^ twist) << 4), to[i][1] = row + (sub >> 2) * kKeyChunk + (((unit + 1) ^ twist) << 4);
            to_rotary[i] = row + 7 * kKeyChunk + (((rotary_sub >> 1) ^ twist) << 4) + 8 * (sub & 1);
        }
        int stage = 0;
        uint32_t stage_at = 0;
        uint32_t phase = 1;  // of kv_empty[stage]: the first round finds it "complete"
        for (int it = 0;; ++it) {
            const int entry = it & 1;
            if (!warp_wait(&rest.look_full[entry], (it >> 1) & 1, limit)) break;
            const uint64_t exist = rest.exist[entry];
            if (exist >> 63) break;
            const uint32_t valid = static_cast<uint32_t>(exist >> (kWarpKeys * reader)) & 0xfu;
            const bool mixed = rest.mixed[entry] != 0;
            ulonglong2 at[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) at[i] = rest.keys[entry][key_a + 2 * i];
            __syncwarp();
            if (lane == 0) barrier_arrive(&rest.look_empty[entry]);
            Values low[2], high[2];
            uint2 rotary[2], codes[2];  // (the code words of `low` and of `high`)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint8_t* data = reinterpret_cast<const uint8_t*>(at[i].x);
                if constexpr (MX) {
                    const uint32_t* code = reinterpret_cast<const uint32_t*>(at[i].y) + (sub >> 3);
                    codes[i] = make_uint2(__ldg(code), __ldg(code + 2));
                    low[i] = ld_stream8(data + 8 * sub);
                    if (coded) high[i] = ld_stream8(data + 128 + 8 * sub);
                    rotary[i] = __ldg(reinterpret_cast<const uint2*>(data + kMxNopeBytes + 8 * rotary_sub));
                } else {
                    codes[i] = __ldg(reinterpret_cast<const uint2*>(at[i].y));
                    low[i] = ld_stream16(data + 16 * sub);
                    if (coded) high[i] = ld_stream16(data + 256 + 16 * sub);
                    rotary[i] = __ldg(reinterpret_cast<const uint2*>(data + kNopeDim + 8 * rotary_sub));
                }
            }
            if (!warp_wait(&rest.kv_empty[stage], phase, limit)) break;
            uint32_t none = ~valid;  // keys of this warp that are stored as zeros
            if (mixed) {
                // Keys that some rows of the tile do not see: those with a value that is not finite are stored as zeros, which the rows that do
                // not see them multiply by zero; the others get NaN as their score.
                uint32_t bad = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint4 a, b;
                    convert(low[i], codes[i].x, a, b);
                    bool any = not_finite(a) || not_finite(b) || not_finite(rotary[i].x) || not_finite(rotary[i].y);
                    if (coded) {
                        convert(high[i], codes[i].y, a, b);
                        any = any || not_finite(a) || not_finite(b);
                    }
                    if (any) bad |= 1u << (2 * i + odd);
                }
                bad = __reduce_or_sync(0xffffffffu, bad) & valid;
                if (lane == 0) rest.bad[stage][reader] = static_cast<uint8_t>(bad);
                none |= bad;
            }
            if ((none & 0xfu) != 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if ((none >> (2 * i + odd)) & 1u) low[i] = high[i] = Values{}, rotary[i] = codes[i] = make_uint2(0u, 0u);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint4 a, b;
                convert(low[i], codes[i].x, a, b);
                store_shared16(to[i][0] + stage_at, a);
                store_shared16(to[i][1] + stage_at, b);
                if (coded) {
                    convert(high[i], codes[i].y, a, b);
                    store_shared16(to[i][0] + stage_at + 4 * kKeyChunk, a);
                    store_shared16(to[i][1] + stage_at + 4 * kKeyChunk, b);
                }
                asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(to_rotary[i] + stage_at), "r"(rotary[i].x), "r"(rotary[i].y) : "memory");
            }
            if (reader == 0 && lane == 0) rest.valid[stage] = exist;
            fence_to_async();
            __syncwarp();
            if (lane == 0) barrier_arrive(&rest.kv_full[stage]);
            stage_at += kKeyBytes;
            if (++stage == kStages) stage = 0, stage_at = 0, phase ^= 1;
        }
    } else if (warp == kIssuerWarp) {
        // ------------------------------------------------------------------------------------------------ products
        if (elected()) {
            bool ok = true;
            int it = 0, tiles = 0, stage = 0, stage_before = 0;
            uint32_t phase = 0, phase_next = 0;
            int stage_next = 0;
            // Barriers are looked at while products are issued: a look takes some 200 cycles in which nothing else is, and the queue of products is short.  (Ahead | not:
            // a block of the chunk 2110 | 2190 cycles; 4 bits, 3.12 | 3.15 ms, 509 listed tokens 370 | 374 us; e4m3, 3.22 | 3.28 ms, window of 512 436 | 443 us, but 61 and 509 listed
            // tokens 25.3 | 24.7 and 381 | 376 us: there the keys are mostly late, and the look is one more.)
            const bool look_ahead = MX || !p.a.indices;
            uint32_t keys_there = 0;
            const auto product_o = [&](int i, bool first, int tile, uint32_t there) {  // O += P V of block i, the one before the last; `there`: P has been seen
                const int buffer = i & 1;
                if (there == 0 && !barrier_wait(&rest.p_full[buffer], (i >> 1) & 1, limit)) return false;
                if (first && tile > 0 && !barrier_wait(&rest.o_empty, (tile - 1) & 1, limit)) return false;
                fence_tmem_after();
                const uint64_t a = operand(base + kOffsetP + buffer * kQueryChunk, 16);
                const uint64_t b = operand(base + kOffsetKeys + stage_before * kKeyBytes, kKeyChunk);
                keys_there = look_ahead ? barrier_test(&rest.kv_full[stage_next], phase_next) : 0u;
#pragma unroll
                for (int half = 0; half < 2; ++half)
#pragma unroll
                    for (int k = 0; k < kBlockKeys / 16; ++k)
                        multiply(tmem + (static_cast<uint32_t>(16 * half) << 16), a + k * (32 >> 4), b + (half * 4 * kKeyChunk + k * 2048) / 16, kKindO,
                                 !first || k > 0);
                commit_to(&rest.kv_empty[stage_before]);
                commit_to(&rest.pv_done[buffer]);
                return true;
            };
            bool pending = false, pending_first = false;
            int pending_tile = 0;
            for (; ok && w.settle(p); w.step(p)) {
                if (w.begin == w.end) continue;
                // (q of this tile is on its way while the last product of the one before runs)
                stage_next = stage, phase_next = phase;
                if (pending && !product_o(it - 1, pending_first, pending_tile, 0)) break;
                pending = false;
                if (!barrier_wait(&rest.q_full, tiles & 1, limit)) break;
                for (int block = w.begin; block < w.end; ++block, ++it) {
                    const int buffer = it & 1;
                    ok = keys_there != 0 || barrier_wait(&rest.kv_full[stage], phase, limit);
                    if (!ok) break;
                    keys_there = 0;
                    fence_tmem_after();
                    const uint64_t a = operand(base, 16), b = operand(base + kOffsetKeys + stage * kKeyBytes, 16);
                    uint32_t p_there = 0;
#pragma unroll
                    for (int chunk = 0; chunk < 8; ++chunk) {
                        if (chunk == kLookChunk) p_there = look_ahead && pending ? barrier_test(&rest.p_full[buffer ^ 1], ((it - 1) >> 1) & 1) : 0u;
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            multiply(tmem_scores + 64 * buffer, a + (chunk * kQueryChunk + 32 * k) / 16, b + (chunk * kKeyChunk + 32 * k) / 16, kKindS,
                                     chunk + k > 0);
                    }
                    commit_to(&rest.s_full[buffer]);
                    if (block + 1 == w.end) commit_to(&rest.q_empty);
                    stage_next = stage + 1 == kStages ? 0 : stage + 1, phase_next = stage + 1 == kStages ? phase ^ 1 : phase;
                    if (pending) ok = product_o(it - 1, pending_first, pending_tile, p_there);
                    if (!ok) break;
                    pending = true, pending_first = block == w.begin, pending_tile = tiles;
                    stage_before = stage;
                    stage = stage_next, phase = phase_next;
                }
                ++tiles;
            }
            if (ok && pending) product_o(it - 1, pending_first, pending_tile, 0);
            // nothing of this CTA may be in flight when its memory is given back, whatever the limit of the other waits
            commit_to(&rest.drained);
            for (uint32_t i = 0; i < kMostWaitRetries && !barrier_try(&rest.drained, 0); ++i) {}
        }
        __syncwarp();
    } else if (warp == kLookupWarp) {
        // ------------------------------------------------------------------------------------------------ look-ups
        // Keys lane and lane + 32 of each block.  Keys that do not exist are given q as their place, and zeroed when they have been read.
        bool ok = true;
        int it = 0;
        const int64_t codes_from = static_cast<int64_t>(p.a.block_size) * kDataBytes;
        for (; ok && w.settle(p); w.step(p)) {
            const Tile& t = w.tile;
            for (int block = w.begin; block < w.end; ++block, ++it) {
                const int entry = it & 1;
                uint64_t exist = 0;
                ulonglong2 at[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int n = lane + 32 * i, k = block * kBlockKeys + n;
                    int number = -1;
                    uint32_t in_block = 0;
                    if (n < kBlockKeys && k < t.keys) {
                        if (p.a.indices) {
                            const int slot = __ldg(p.a.indices + t.token * p.a.indices_stride + k);
                            if (slot >= 0) {
                                number = fast_div(slot, p.a.block_mul, p.a.block_shift);
                                in_block = slot - static_cast<uint32_t>(number) * p.a.block_size;
                            }
                        } else {
                            const uint32_t where = k < t.first ? k : k - t.first + t.low, page = fast_div(where, p.a.block_mul, p.a.block_shift);
                            in_block = where - page * p.a.block_size;
                            number = __ldg(p.a.block_table + w.at.request * p.a.table_stride + page);
                        }
                    }
                    const bool there = number >= 0 && number < p.a.num_blocks;
                    const uint8_t* block_at = p.a.k_cache + number * p.a.block_stride;
                    at[i].x = reinterpret_cast<uint64_t>(there ? block_at + static_cast<int64_t>(in_block) * kDataBytes : p.a.q);
                    at[i].y = reinterpret_cast<uint64_t>(there ? block_at + codes_from + static_cast<int64_t>(in_block) * kCodeBytes : p.a.q);
                    exist |= static_cast<uint64_t>(__ballot_sync(0xffffffffu, there)) << (32 * i);
                    // A key's record goes to L2 two blocks before a reader asks for it (61 requests of up to 16384 keys: 116.0 -> 110.6 us).  The keys of
                    // a page lie one behind the other, so three lines of each are all of its 22.5 KB; listed keys gain nothing (509 tokens: 369 -> 379 us).
                    if (MX && there && !p.a.indices) {
                        const uint8_t* record = reinterpret_cast<const uint8_t*>(at[i].x);
#pragma unroll
                        for (int line = 0; line < 3; ++line) prefetch_line_l2(record + 128 * line);
                        if ((lane & 7) == 0) prefetch_line_l2(reinterpret_cast<const uint8_t*>(at[i].y));
                    }
                }
                ok = warp_wait(&rest.look_empty[entry], ((it >> 1) - 1) & 1, limit);
                if (!ok) break;
                rest.keys[entry][lane] = at[0];
                if (lane + 32 < kBlockKeys) rest.keys[entry][lane + 32] = at[1];
                if (lane == 0) rest.exist[entry] = exist, rest.mixed[entry] = t.mixed(p, block);
                __syncwarp();
                if (lane == 0) barrier_arrive(&rest.look_full[entry]);
            }
        }
        // the end
        ok = ok && warp_wait(&rest.look_empty[it & 1], ((it >> 1) - 1) & 1, limit);
        if (ok && lane == 0) rest.exist[it & 1] = 1ull << 63, barrier_arrive(&rest.look_full[it & 1]);
    } else {
        // ------------------------------------------------------------------------------------------------ queries
        int tiles = 0;
        for (; w.settle(p); w.step(p)) {
            if (w.begin == w.end) continue;
            const Tile& t = w.tile;
            if (tiles > 0 && !warp_wait(&rest.q_empty, (tiles - 1) & 1, limit)) break;
            // Atoms of eight rows in turn; a row is 64 pieces of 16 bytes, two passes of the warp.  (These warps share their schedulers with the
            // readers: the time that a tile's queries take is that of the instructions for them.)
            const int own = warp - kLookupWarp - 1;
            int row = 8 * own, token = t.token, head = t.head + row;
#pragma unroll 1
            for (; row < kRows; row += 8 * (kQueryWarps - 1), head += 8 * (kQueryWarps - 1)) {
                if (t.count > 1) token = t.token + row / p.a.num_heads, head = row % p.a.num_heads;
                const uint8_t* from = p.a.q + token * p.a.q_stride_token + head * p.a.q_stride_head + 16 * lane;
                const uint32_t to = base + (lane >> 3) * kQueryChunk + row * 128;
#pragma unroll
                for (int i = 0; i < 8; ++i, ++row) {
                    const uint32_t at = to + i * 128 + (((lane & 7) ^ i) << 4);
                    const bool live = row < t.rows;
                    const uint8_t* safe = live ? from : p.a.q;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(safe), "r"(live ? 16 : 0) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + 4 * kQueryChunk), "l"(safe + 512), "r"(live ? 16 : 0) : "memory");
                    from += p.a.q_stride_head;
                    if (++head == p.a.num_heads && t.count > 1) head = 0, from += p.a.q_stride_token - p.a.num_heads * p.a.q_stride_head;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_to_async();
            __syncwarp();
            if (lane == 0) barrier_arrive(&rest.q_full);
            ++tiles;
        }
    }
    fence_tmem_before();
    __syncthreads();
    if (warp == kIssuerWarp) {
        fence_tmem_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    }
}

// Joins the pieces of tiles that were cut, which the CTAs of the kernel above have left in order: the head of a tile in one CTA, the rest in the
// CTAs behind it.  A CTA takes rows in turn, one warp a row, or 4 or 16 warps that share out the pieces of a row where there are many.  (A CTA for
// every row that might need it took 15 to 28 us, most of it for those that did not.)
constexpr int kJoinWarps = 16, kJoinCtas = 2 * kMaxCtas;
__global__ void __launch_bounds__(kJoinWarps * 32) join_pieces_kernel(const Launched<Tiles> p) {
    begin_dependent_kernel();
    __shared__ int4 pieces[2 * kMaxCtas];
    __shared__ int heads[kMaxCtas], ends[kMaxCtas], counts[2][kJoinWarps], most;
    __shared__ float4 part[kJoinWarps][kHeadDim / 4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int i = tid; i < 2 * kMaxCtas; i += kJoinWarps * 32) pieces[i] = p.pieces[i];
    if (tid < kMaxCtas) ends[tid] = -1;
    if (tid == 0) most = 0;
    __syncthreads();
    // The tiles: the CTA with the head and the one with the end of each, which follow one another.
    const bool head = tid < kMaxCtas && pieces[2 * tid + 1].w != 0, end = tid < kMaxCtas && pieces[2 * tid].w == 2;
    const uint32_t head_votes = __ballot_sync(0xffffffffu, head), end_votes = __ballot_sync(0xffffffffu, end);
    if (lane == 0) counts[0][warp] = __popc(head_votes), counts[1][warp] = __popc(end_votes);
    __syncthreads();
    int tiles = 0, heads_before = __popc(head_votes & ((1u << lane) - 1u)), ends_before = __popc(end_votes & ((1u << lane) - 1u));
    for (int w = 0; w < kJoinWarps; ++w) {
        if (w < warp) heads_before += counts[0][w], ends_before += counts[1][w];
        tiles += counts[0][w];
    }
    if (head) heads[heads_before] = tid;
    if (end) ends[ends_before] = tid;
    __syncthreads();
    // Heads and ends pair up in order, unless a wait of the kernel above ran out: a CTA that gave up has left no record of one or the other.  A head keeps its
    // end only where that lies behind it, before the next head's CTA or in it, and is of the same tile; a tile without one is left as it was.
    if (tid < tiles) {
        const int from = heads[tid], to = ends[tid], most_to = tid + 1 < tiles ? heads[tid + 1] : kMaxCtas - 1;
        const bool pair = to > from && to <= most_to && pieces[2 * to].x == pieces[2 * from + 1].x && pieces[2 * to].y == pieces[2 * from + 1].y;
        if (pair) atomicMax(&most, to - from + 1);
        else ends[tid] = -1;
    }
    __syncthreads();
    const int each = most <= 4 ? 1 : most <= 16 ? 4 : 16, rows = kJoinWarps / each, turn = warp % each;  // warps for a row, rows at once
    const float c = p.a.scale * kLog2e;
    constexpr int kPerLane = (kMaxCtas + 31) / 32;
    for (int item = blockIdx.x; item < tiles * (kRows / rows); item += kJoinCtas) {
        const int tile = item / (kRows / rows), row = item % (kRows / rows) * rows + warp / each;
        const int first = heads[tile], count = ends[tile] - first + 1;
        if (ends[tile] < 0) continue;  // (the same for the whole CTA)
        const int4 of = pieces[2 * first + 1];
        const bool live = row < of.z;
        // piece i: that of CTA first + i, where it has one
        const auto slot_of = [&](int i) { return i == 0 ? 2 * first + 1 : pieces[2 * (first + i)].w != 0 ? 2 * (first + i) : -1; };
        float2 state[kPerLane];
        float m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
            const int i = lane + 32 * k, slot = live && i < count ? slot_of(i) : -1;
            state[k] = slot >= 0 ? p.rows[slot * kRows + row] : make_float2(-INFINITY, 0.0f);
            m = fmaxf(m, state[k].x);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
            const bool some = state[k].x != -INFINITY;
            state[k].x = some ? exp2_approx((state[k].x - m) * c) : 0.0f;
            l += some ? state[k].y * state[k].x : state[k].y;  // (a sum that is NaN stays NaN, also that of a row without a finite maximum)
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        float4 o[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) {
#pragma unroll 2
            for (int i = 32 * k + turn; i < min(count, 32 * k + 32); i += each) {
                const float f = __shfl_sync(0xffffffffu, state[k].x, i & 31);
                const int slot = slot_of(i);
                if (slot < 0 || !live) continue;
                const float4* from = reinterpret_cast<const float4*>(p.sums + (static_cast<int64_t>(slot) * kRows + row) * kHeadDim) + lane;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 v = __ldg(from + 32 * q);
                    o[q].x = fmaf(v.x, f, o[q].x), o[q].y = fmaf(v.y, f, o[q].y), o[q].z = fmaf(v.z, f, o[q].z), o[q].w = fmaf(v.w, f, o[q].w);
                }
            }
        }
        const int token = of.x + (p.head_groups == 1 ? row / p.a.num_heads : 0), at = p.head_groups == 1 ? row % p.a.num_heads : of.y + row;
        const bool some = l != 0.0f;
        float total = l;
        if (live && p.a.sink && some) total += exp2_approx(fmaf(__ldg(p.a.sink + at), kLog2e, -m * c));
        const float inverse = some ? 1.0f / total : 0.0f;
        const auto store = [&](int dim, const float4& v) {  // of four dimensions
            *reinterpret_cast<uint2*>(p.a.out + token * p.a.out_stride_token + at * p.a.out_stride_head + 8 * dim) =
                some ? make_uint2(pack_bf16x2(v.x * inverse, v.y * inverse), pack_bf16x2(v.z * inverse, v.w * inverse)) : make_uint2(0u, 0u);
        };
        if (live && turn == 0 && lane == 0 && p.a.lse)
            p.a.lse[token * p.a.lse_stride_token + at * p.a.lse_stride_head] = some ? (m * c + log2f(l)) * kLn2 : -INFINITY;
        if (each == 1) {
            if (live)
                for (int q = 0; q < 4; ++q) store(lane + 32 * q, o[q]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) part[warp][lane + 32 * q] = o[q];
            __syncthreads();
            for (int dim = 32 * turn + lane; live && dim < kHeadDim / 4; dim += 32 * each) {
                float4 sum = part[warp - turn][dim];
                for (int w = 1; w < each; ++w) {
                    const float4 v = part[warp - turn + w][dim];
                    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
                }
                store(dim, sum);
            }
            __syncthreads();
        }
    }
}

constexpr size_t kSumBytes = sizeof(float) * 2 * kMaxCtas * kRows * kHeadDim, kRowBytes2 = sizeof(float2) * 2 * kMaxCtas * kRows;

}  // namespace

size_t latent_attention_workspace(int64_t, int64_t) { return kSumBytes + kRowBytes2 + sizeof(int4) * 2 * kMaxCtas; }

cudaError_t launch_latent_attention(const LatentAttention& a, bool mxfp4, void* workspace, cudaStream_t stream) {
    const auto kernel = mxfp4 ? latent_attention_kernel<true> : latent_attention_kernel<false>;
    Tiles p{};
    p.a = a;
    p.lists = Lists{a.query_start_loc, a.indices ? a.lens : a.seq_lens};
    p.tokens_per_tile = a.indices || a.num_heads >= kRows ? 1 : kRows / a.num_heads;
    p.head_groups = (a.num_heads + kRows - 1) / kRows;
    const int64_t most_keys = a.indices ? a.topk : std::min<int64_t>(a.capacity, a.window > 0 ? static_cast<int64_t>(a.window) + a.first + p.tokens_per_tile : a.capacity);
    const int64_t most_blocks = (most_keys + kBlockKeys - 1) / kBlockKeys, tiles = static_cast<int64_t>(a.num_tokens) * p.head_groups;
    const int64_t fewest_tiles = (static_cast<int64_t>(a.num_tokens) + p.tokens_per_tile - 1) / p.tokens_per_tile * p.head_groups;
    p.one_each = tiles <= kMaxCtas && (most_blocks < kLeastSplit || (most_blocks <= kMostWhole && most_blocks * (kMaxCtas - fewest_tiles) <= kSplitCost * kMaxCtas));
    const bool may_split = !p.one_each && most_blocks >= kLeastSplit;
    auto* at = static_cast<uint8_t*>(workspace);
    p.sums = reinterpret_cast<float*>(at), p.rows = reinterpret_cast<float2*>(at + kSumBytes), p.pieces = reinterpret_cast<int4*>(at + kSumBytes + kRowBytes2);
    // A setmaxnreg that asks for more than the block was launched with waits forever, and how many that is the compiler chooses: looked at once for each kernel.
    const auto as_expected = [](auto* of) {
        cudaFuncAttributes a;
        const cudaError_t error = cudaFuncGetAttributes(&a, of);
        return error != cudaSuccess ? error : a.numRegs == kLaunchRegisters ? cudaSuccess : cudaErrorLaunchOutOfResources;
    };
    static std::atomic<bool> looked[2] = {};
    if (!looked[mxfp4].load(std::memory_order_relaxed)) {
        const cudaError_t rc = as_expected(kernel);
        if (rc != cudaSuccess) return rc;
        looked[mxfp4].store(true, std::memory_order_relaxed);
    }
    // Set for the current device each time: cheaper than to remember for which ones it was.
    cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes);
    if (rc != cudaSuccess) return rc;
    rc = launch_dependent_cluster(kernel, dim3(kMaxCtas), dim3(kThreads), 1, kSharedBytes, stream, p);
    if (rc != cudaSuccess) return rc;
    count_launch();
    if (!may_split) return cudaGetLastError();
    rc = launch_dependent(join_pieces_kernel, dim3(kJoinCtas), dim3(kJoinWarps * 32), stream, p);
    if (rc != cudaSuccess) return rc;
    count_launch();
    return cudaGetLastError();
}

cudaError_t read_attention_error(int* value) {
    int zero = 0;
    const cudaError_t rc = cudaMemcpyFromSymbol(value, g_attention_error, sizeof(int));
    return rc != cudaSuccess || *value == 0 ? rc : cudaMemcpyToSymbol(g_attention_error, &zero, sizeof(int));
}

}  // namespace dsv4
