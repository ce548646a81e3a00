// Attention of many new tokens over the 8-bit paged cache (kv8.cuh) on the 5th-generation tensor cores: causal, optionally
// windowed, grouped query heads, runs of unequal length packed back to back.  Heads of up to 128 channels.
//
//   S = Q K^T      tcgen05.mma, 128 queries by 128 keys, accumulated in 32-bit in tensor memory
//   P = 2^(S log2(e) / sqrt(hd) - m)   in 32-bit, by two threads a row; rounded to bfloat16 and written over S, where the next
//                  product reads it as its A operand
//   O += P V       tcgen05.mma, accumulated in tensor memory
//
// m is a whole number near the row's running maximum, which may have outgrown it by 2^LAZY: only then are O and the row's sum scaled anew.
// Scores are good below 2^30 in units of log2: above it m, rounded to 32 bits, is off from the maximum by as much as a weight's exponent has
// room for, and a row may be NaN.  (Rounding such scores first, behind a test of m for every 32 of them, cost 7 % of the ragged chunks
// below; the streaming kernels have no such bound.)
//
// The cache's codes cannot be operands beside bfloat16 queries and weights, so eight warps turn them into bfloat16 on their way
// from global to shared memory: a code's bits moved into a bfloat16's places are the code times 2^-120, subnormal codes
// included, and one multiplication by 2^(120 + e) gives the number exactly.  That is four operations for two codes,
// 2.4 with loads and stores for each, against about 3.5 of the row threads for each score.  A block of keys is therefore made
// once for 256 queries: an item is two tiles of 128 new tokens of a sequence (PAIR), each with a group of row threads and S and O
// of its own, in all 512 columns of tensor memory.  Where there are few items, or a tile has no neighbour, the two groups
// take the blocks of one tile in turn instead (SPLIT) and join their results.
//
// Measured (B200): 8,192 tokens, 16 heads of 128, 280 to 300 us in runs of 20 calls and 306 in long ones, whose clocks are lower (0.98 to
// 0.90 PFLOP/s; the kernel for the bfloat16 cache 335 in short runs); five ragged chunks of 500 to 1,500 tokens behind contexts of
// 1,500 to 4,600, 28 heads on 4, 395 and 415 us (0.88, 0.84).  A step of one block for both tiles takes about
// 4,000 cycles, of which the tensor core needs 2,050 (counters: tensor pipe 48 %, issue slots 63 %, ALU 49 %, exponentials 50 %).  What
// bounds it are the converting warps (their loads and stores share shared memory's 128 bytes a cycle with the MMAs' operands, their
// instructions the issue slots with the row threads) and, close behind, a group's chain: scores, weights and meeting 2,200 cycles, then
// P V and the next scores 1,024.  An item costs about 5 us besides (its first and last products and its results, which nothing of the
// same rows overlaps).  Spills cost more than anything else: beside 200 KB of shared memory they miss L1 (17 local loads a warp and
// block: 393 us for 296).
//
// Keys of a page that is none have no weight, as in the streaming kernels: the row threads, each of which has the keys of one page of a
// block, look it up where the item meets such a page.  A row without keys is zeros.
//
// A position that is no number (kv8.cuh) is made a key of NaN with a value of zeros: whoever sees it gets NaN through the score,
// and a masked score takes nothing of it.
//
// Every wait is bounded, and a warp whose wait runs out leaves, row threads once they have been at the meetings where others would
// wait for them without a limit (kv8_walk.cuh); the waits that hang on it then run out too.  (A flag that every wait looks at first
// cost 8 of 291 us.)
#include "kv8.cuh"
#include "kv8_walk.cuh"
#include "tc05.cuh"

namespace {
using namespace tc05;
constexpr int BM = 128, BN = 128, ATOM = 128 * 128;     // ATOM: bytes of a 64-channel slice of 128 rows
constexpr int STAGES = 2;                               // blocks of keys (and of values) in shared memory as bfloat16
// warps: 0-7 and 8-15 the groups of row threads (two threads a row), 16-23 codes to bfloat16, 24 MMA, 25 queries, 26 pages and
// exponents, 27 none.  Registers are moved between them (whole groups of four warps): 512 * 80 + 256 * 56 + 128 * 72 = 64,512,
// the launch's 896 * 72.
constexpr int ROW_WARPS = 16, CONV_WARPS = 8, MMA_WARP = 24, Q_WARP = 25, PAGE_WARP = 26, THREADS = 896;
constexpr int AHEAD = 4;                                // blocks of keys whose pages and exponents are known ahead
constexpr int LIST = 4096;                              // tiles of a launch
constexpr int FEW = 1024;                               // tiles of a launch that looks which way is better
enum { SINGLY, IN_PAIRS, LOOK };                        // ways of a launch
constexpr unsigned LIST_PAIR = 0x8000;                  // of a list's entry: the tile takes the next of its sequence along
constexpr float LAZY = 8.f;
// Values are taken times 2^-V_DOWN and results times 2^V_DOWN, so that sums of weights of up to 2^LAZY times values of up to 448 * 2^100
// stay in 32-bit's range for 2^23 keys; a value's smallest code, 2^-109, still is a normal bfloat16.
constexpr int V_DOWN = 12;

struct Params {
    const unsigned char *k, *v, *exps;
    bf16* out;
    const int *tile_seq, *tile_first, *seq_start, *seq_past, *block_table;
    int n_seqs, table_stride, n_pages, nh, nkv, hd, window, n_tiles;
    short way, least;                                   // shorts: an int more here and the compiler spills in the row threads' loop (2 %)
    int smem_bytes, n_tokens;
    float scale_log2;
    int* status;
};

__host__ __device__ constexpr unsigned idesc_attn(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? (1u << 16) : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
}
// Operand descriptors (128-byte swizzle, groups of 8 rows 1,024 bytes apart): the high word is the same for all, the low word
// holds the address and, for an MN-major operand (rows are keys, 128 bytes of channels each), how far the next 64
// channels lie.
constexpr unsigned DESC_HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ unsigned desc_low(unsigned addr, unsigned next) { return ((addr & 0x3FFFFu) >> 4) | (next >> 4) << 16; }
// D += A B with A in tensor memory
__device__ __forceinline__ void tc_mma_ta_lo(unsigned tmem_d, unsigned tmem_a, unsigned b_lo, unsigned idesc, unsigned accumulate) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 db;\n"
        "setp.ne.b32 p, %5, 0;\n"
        "mov.b64 db, {%2, %3};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(DESC_HIGH), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    unsigned r;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// two numbers by one instruction: (a, b) * m + c, and sum + (a, b)
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 parts_of(unsigned long long x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ unsigned long long fma_pair(unsigned long long a, unsigned long long m, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(m), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add_pair(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ bool all_agree(bool ok, int id, int count) {
    unsigned all;
    asm volatile(
        "{\n.reg .pred p, q;\n"
        "setp.ne.u32 p, %1, 0;\n"
        "bar.red.and.pred q, %2, %3, p;\n"
        "selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(all) : "r"(ok ? 1u : 0u), "r"(id), "r"(count) : "memory");
    return all != 0;
}
__device__ __forceinline__ void named_sync(int id, int count) { asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(count) : "memory"); }
// 32 consecutive columns of this thread's lane, asked for; tc_wait_ld() before they are used
__device__ __forceinline__ void tc_ask32(unsigned taddr, unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_ld8(unsigned taddr, unsigned (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])::"memory");
}
__device__ __forceinline__ void tc_st8(unsigned taddr, const unsigned (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// the loads have arrived: their registers pass through here, so that no use is moved ahead of the wait
__device__ __forceinline__ void tc_wait_ld(unsigned (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
          "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
          "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
          "+r"(r[31])::"memory");
}

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    __nv_bfloat162 w = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<unsigned*>(&w);
}

// ---- two codes' bits (two bytes of w) in a bfloat16 pair's places: each is its number times 2^-120
template <unsigned SELECT> __device__ __forceinline__ unsigned spread_codes(unsigned w) {
    unsigned r;                                         // bytes (code, its sign eight times) of two codes
    asm("prmt.b32 %0, %1, %1, %2;\n" : "=r"(r) : "r"(w), "n"(SELECT));
    return (r << 4) & 0x87f087f0u;
}
__device__ __forceinline__ unsigned mul_bf16x2(unsigned a, unsigned b) {
    unsigned r;
    asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// What the converting warps are told of a block of keys: its two pages' places in the pools ((page * nkv + head), -1: none), the
// rows that exist for the item, and the exponents of the pages' keys and values.
template <int R> struct Word;
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<2> { typedef unsigned short type; };
struct Entry {
    int block[2], lo, hi;                               // hi -1: no more work
    unsigned char exps[2][2][KV8_PAGE];
};
// What a block works on: one or two tiles of 128 query rows of a head.
struct Item {
    int seq, h, kvh, row0, first, news, past, blk0, nb, key_lo, key_hi;
    bool pair;
    __device__ __forceinline__ int rows(int g) const { return min(BM, news - first - (pair ? g * BM : 0)); }
    __device__ __forceinline__ int pos0(int g) const { return past + first + (pair ? g * BM : 0); }
    // a tile's blocks of keys, counted from blk0
    __device__ __forceinline__ int lo(int g, int window) const { return first_visible_key(pos0(g), window, 0) / BN - blk0; }
    __device__ __forceinline__ int hi(int g) const { return (pos0(g) + rows(g) - 1) / BN - blk0; }
};
__device__ __forceinline__ Item load_item(const Params& p, const unsigned short* list, int item) {
    Item t;
    const unsigned entry = list[item / p.nh], tile = entry & (LIST_PAIR - 1);
    t.h = item % p.nh;
    t.kvh = t.h / (p.nh / p.nkv);
    t.seq = p.tile_seq[tile];
    const int start = p.seq_start[t.seq];
    t.first = p.tile_first[tile];
    t.news = p.seq_start[t.seq + 1] - start;
    t.past = p.seq_past[t.seq];
    t.row0 = start + t.first;
    t.pair = entry & LIST_PAIR;
    t.key_lo = first_visible_key(t.pos0(0), p.window, 0);
    t.key_hi = t.pos0(1) + t.rows(1) - 1;
    t.blk0 = t.key_lo / BN;
    t.nb = t.key_hi / BN - t.blk0 + 1;
    return t;
}

// whether the sequence's page of position ``key`` is one; whether that of any of the positions lo .. hi is
__device__ __forceinline__ bool has_page(const int* table, int table_stride, int n_pages, int seq, int key) {
    const int i = key / KV8_PAGE, page = i < table_stride ? table[(size_t)seq * table_stride + i] : -1;
    return page >= 0 && page < n_pages;
}
__device__ __noinline__ bool has_pages(const int* table, int table_stride, int n_pages, int seq, int lo, int hi) {
    for (int i = lo / KV8_PAGE; i <= hi / KV8_PAGE; i++)
        if (has_page(table, table_stride, n_pages, seq, i * KV8_PAGE)) return true;
    return false;
}

// a warp: whether one of them is none
__device__ __forceinline__ bool misses_page(const int* table, int table_stride, int n_pages, int seq, int lo, int hi, int lane) {
    bool misses = false;
#pragma unroll 4
    for (int i = lo / KV8_PAGE + lane; i <= hi / KV8_PAGE; i += 32) misses |= !has_page(table, table_stride, n_pages, seq, i * KV8_PAGE);
    return __any_sync(0xffffffffu, misses);
}

template <int HD>
__global__ void __launch_bounds__(THREADS, 1) attn_prefill_kv8_kernel(const __grid_constant__ CUtensorMap map_q, const Params p) {
    constexpr int HALVES = HD / 64, TILE = HALVES * ATOM;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* q_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);   // [2]
    unsigned char* k_s = q_s + 2 * TILE;                 // [STAGES]
    unsigned char* v_s = k_s + STAGES * TILE;            // [STAGES]
    unsigned long long* bars = reinterpret_cast<unsigned long long*>(v_s + STAGES * TILE);
    unsigned long long *q_full = bars, *q_empty = bars + 1, *drained = bars + 2, *s_full = bars + 4, *p_ready = bars + 6, *o_full = bars + 8,
                       *o_free = bars + 10, *k_full = bars + 12, *k_empty = k_full + STAGES, *v_full = k_empty + STAGES, *v_empty = v_full + STAGES,
                       *e_full = v_empty + STAGES, *e_empty = e_full + AHEAD;
    constexpr int N_BARS = 12 + 4 * STAGES + 2 * AHEAD;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + N_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* n_listed = reinterpret_cast<int*>(tmem_slot + 2);       // [2]: pairs, tiles
    int* longest = n_listed + 2;                         // [2]: the time of the block with the most work, in pairs and singly
    float* xmax = reinterpret_cast<float*>(bars + 36);   // [group][parity][side][row]: maxima of a block
    float* xsum = xmax + 2 * 2 * 2 * 128;                // [group][side][row]: sums at the item's end
    float* xref = xsum + 2 * 2 * 128;                    // [group][row]: the maxima that they go with
    Entry* entries = reinterpret_cast<Entry*>(xref + 2 * 128);           // [AHEAD]
    unsigned short* list = reinterpret_cast<unsigned short*>(entries + AHEAD);       // of the tiles that begin a pair
    // where they are few: of all tiles, and [2][FEW] the blocks of keys of both lists' entries (before there are keys)
    unsigned short *singles = list + FEW, *steps = reinterpret_cast<unsigned short*>(k_s);
    static_assert(N_BARS <= 32, "the barriers and six words take 288 bytes");
    if (reinterpret_cast<unsigned char*>(list + LIST) > smem_raw + p.smem_bytes) {
        if (threadIdx.x == 0) atomicOr(p.status, ESP_STATUS_SMEM_LAYOUT);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < N_BARS; i++) mbar_init(&bars[i], 1);
        for (int g = 0; g < 2; g++) {
            mbar_init(&p_ready[g], 8);                   // a warp of the group's rows each
            mbar_init(&o_free[g], 8);
        }
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&k_full[s], CONV_WARPS);
            mbar_init(&v_full[s], CONV_WARPS);
        }
        for (int s = 0; s < AHEAD; s++) mbar_init(&e_empty[s], CONV_WARPS);
        *abort_flag = 0;
        longest[0] = longest[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    pdl_wait();
    pdl_trigger();
    // ---- the tiles that begin an item, in the order of the list: singly all, with pairs those whose place in their sequence is even
    if (warp == Q_WARP) {
        int n = 0, n_pairs = 0;
        for (int i0 = 0; i0 < p.n_tiles; i0 += 32) {
            const int i = i0 + lane;
            bool fine = false, begins = false, goes_on = false;
            int blocks = 0, both = 0;
            if (i < p.n_tiles) {
                // a tile of a sequence that is not there, that is none of its tiles, without rows or with rows that the queries do not have, or with positions that the
                // page table does not have is left out
                const int seq = p.tile_seq[i], first = p.tile_first[i];
                fine = seq >= 0 && seq < p.n_seqs && first >= 0 && first % BM == 0;
                if (fine) {
                    const int start = p.seq_start[seq], end = p.seq_start[seq + 1], past = p.seq_past[seq];
                    fine = start >= 0 && end >= start && end <= p.n_tokens && first < end - start && past >= 0 &&
                           ((long long)past + (end - start) - 1) / KV8_PAGE < p.table_stride;
                    const int pos = past + first, lo = first_visible_key(pos, p.window, 0) / BN, last = past + end - start - 1;
                    if (!fine && blockIdx.x == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
                    fine = fine && end - start >= p.least;               // the others are another kernel's
                    begins = fine && first / BM % 2 == 0;
                    goes_on = first + BM < end - start;
                    blocks = min(pos + BM - 1, last) / BN - lo + 1, both = min(pos + 2 * BM - 1, last) / BN - lo + 1;
                }
                else if (blockIdx.x == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
            }
            const unsigned below = (1u << lane) - 1u, mask = __ballot_sync(0xffffffffu, fine), mask2 = __ballot_sync(0xffffffffu, begins);
            if (fine && p.way != IN_PAIRS) {
                const int at = n + __popc(mask & below);
                (p.way == LOOK ? singles : list)[at] = (unsigned short)i;
                if (p.way == LOOK) steps[FEW + at] = (unsigned short)min(blocks, 65535);
            }
            if (begins && p.way != SINGLY) {
                const int at = n_pairs + __popc(mask2 & below);
                list[at] = (unsigned short)(i | (goes_on ? LIST_PAIR : 0u));
                if (p.way == LOOK) steps[at] = (unsigned short)min(both, 65535);
            }
            n += __popc(mask);
            n_pairs += __popc(mask2);
        }
        if (lane == 0) {
            n_listed[0] = n_pairs;
            n_listed[1] = n;
        }
    }
    const int G = gridDim.x;
    // block b takes the items b, 2G-1-b, 2G+b, ...: a long one is followed by a short one
    auto nth_item = [&](int b, int round) { return round * G + (round & 1 ? G - 1 - b : b); };
    // Pairs halve the conversions but are fewer and longer items, for which a step (a block of keys) takes 4/3 of the time.  Every block
    // works out what the block with the most work has either way, an item counting three steps more than it has.  (210 tiles behind
    // 4,953 keys: 138 us singly, 109 in pairs; 512 of a prompt of 4,096: 108 and 80; 256 of a prompt of 2,048: 37 and 46; 232 of four
    // prompts of 3,693: 58 and 81.)
    if (p.way == LOOK) {
        __syncthreads();
        int most[2] = {0, 0};
        if ((int)threadIdx.x < G) {
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int items = n_listed[u] * p.nh;
                for (int round = 0; round * G < items; round++) {
                    const int item = nth_item(threadIdx.x, round);
                    if (item < items) most[u] += steps[u * FEW + item / p.nh] + 3;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            most[u] = __reduce_max_sync(0xffffffffu, most[u]);
            if (lane == 0 && most[u] > 0) atomicMax(&longest[u], most[u]);
        }
        __syncthreads();
        if (4LL * longest[0] >= 3LL * longest[1]) {
            for (int i = threadIdx.x; i < n_listed[1]; i += THREADS) list[i] = singles[i];
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = (unsigned)uniform((int)*tmem_slot), tm_s = tmem, tm_o = tmem + 256;    // S of the groups at columns 0 and 128, O at 256 and 384
    const int n_items = n_listed[p.way == IN_PAIRS || (p.way == LOOK && 4LL * longest[0] < 3LL * longest[1]) ? 0 : 1] * p.nh;
    auto item_of = [&](int round) { return nth_item(blockIdx.x, round); };

    if (warp >= MMA_WARP) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
    if (warp == Q_WARP) {
        bool ok = true;
        int issued = 0;
        for (int round = 0; ok; round++) {
            const int item = item_of(round);
            if (item >= n_items) break;
            const Item t = load_item(p, list, item);
            const int tiles = t.pair ? 2 : 1;
            if (lane == 0) {
                ok = !*abort_flag && mbar_wait(q_empty, (round & 1) ^ 1);
                if (ok) mbar_expect_tx(q_full, tiles * TILE);
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            if (lane < tiles * HALVES)
                tma_load_3d(q_s + lane * ATOM, &map_q, (lane % HALVES) * 64, t.h, t.row0 + (lane / HALVES) * BM, q_full);
            issued = round + 1;
        }
        if (lane == 0 && (!ok || *abort_flag)) {
            atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
            *abort_flag = 1;
            if (issued > 0) mbar_wait(q_full, (issued - 1) & 1);         // its copies land before the block ends
        }
    } else if (warp == MMA_WARP) {
        // The whole warp walks the blocks, so that what the MMAs are given is known to be the same for all lanes; one of them
        // issues.  S of a block overwrites the P before it, so its group's P V comes first: the tensor core runs one
        // thread's products in the order in which they were issued.
        const bool leader = elect_one();
        constexpr unsigned idesc_s = idesc_attn(BN, false), idesc_pv = idesc_attn(HD, true);
        const unsigned dq = desc_low(smem_u32(q_s), 16), dk = desc_low(smem_u32(k_s), 16), dv = desc_low(smem_u32(v_s), ATOM);
        bool ok = true;
        int b0 = 0;                                                       // key blocks before this item
        unsigned ph_p = 0, ph_o = 0;                                      // a bit a group: the phase of its P, of its O
        for (int round = 0; ok; round++) {
            const int item = item_of(round);
            if (item >= n_items) break;
            const Item t = load_item(p, list, item);
            const int pair = uniform(t.pair), nb = uniform(t.nb), lo0 = uniform(t.lo(0, p.window)), hi0 = uniform(t.hi(0)),
                      lo1 = uniform(t.lo(1, p.window)), hi1 = uniform(t.hi(1));
            ok = __all_sync(0xffffffffu, mbar_wait(q_full, round & 1));
            unsigned begun = 0;                                           // a bit a group: its O holds something of this item
            auto issue_s = [&](const int g, int j, bool last_use, bool last) {
                const int st = (b0 + j) % STAGES;
                if (!__all_sync(0xffffffffu, mbar_wait(&k_full[st], ((b0 + j) / STAGES) & 1))) return false;
                tc_fence_after();
                const unsigned qa = dq + (pair ? (unsigned)(g * TILE) >> 4 : 0u), kb = dk + ((unsigned)(st * TILE) >> 4);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const unsigned off = ((kk >> 2) * ATOM + (kk & 3) * 32) >> 4;
                        tc_mma_lo(tm_s + g * BN, qa + off, kb + off, DESC_HIGH, idesc_s, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(&s_full[g]);
                    if (last_use) tc_commit(&k_empty[st]);
                    if (last) tc_commit(q_empty);
                }
                __syncwarp();
                return true;
            };
            auto issue_pv = [&](const int g, int j, bool last_use, bool last) {
                const int st = (b0 + j) % STAGES;
                // the first P V of an item: the row threads have read the O of the item before
                bool fine = (begun >> g & 1) || mbar_wait(&o_free[g], (ph_o >> g & 1) ^ 1);
                fine = fine && mbar_wait(&v_full[st], ((b0 + j) / STAGES) & 1) && mbar_wait(&p_ready[g], ph_p >> g & 1);
                if (!__all_sync(0xffffffffu, fine)) return false;
                tc_fence_after();
                const unsigned vb = dv + ((unsigned)(st * TILE) >> 4), first = begun >> g & 1;
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < BN / 16; kk++)
                        tc_mma_ta_lo(tm_o + g * BN, tm_s + g * BN + (kk >> 2) * 64 + (kk & 3) * 8, vb + ((kk * 16 * 128) >> 4), idesc_pv, kk > 0 ? 1u : first);
                    if (last_use) tc_commit(&v_empty[st]);
                    if (last) tc_commit(&o_full[g]);
                }
                __syncwarp();
                ph_p ^= 1u << g;
                if (!first) ph_o ^= 1u << g;
                begun |= 1u << g;
                return true;
            };
            if (pair) {
                for (int j = 0; j <= nb && ok; j++) {
                    if (ok && j - 1 >= lo0 && j - 1 <= hi0) ok = issue_pv(0, j - 1, j - 1 < lo1, j - 1 == hi0);
                    if (ok && j >= lo0 && j <= hi0) ok = issue_s(0, j, j < lo1, false);
                    if (ok && j - 1 >= lo1 && j - 1 <= hi1) ok = issue_pv(1, j - 1, true, j - 1 == hi1);
                    if (ok && j >= lo1 && j <= hi1) ok = issue_s(1, j, true, j == hi1);
                }
            } else {
                for (int j = 0; j < nb + 2 && ok; j++) {
                    if (j >= 2) ok = j & 1 ? issue_pv(1, j - 2, true, j >= nb) : issue_pv(0, j - 2, true, j >= nb);
                    if (ok && j < nb) ok = j & 1 ? issue_s(1, j, true, j + 1 == nb) : issue_s(0, j, true, j + 1 == nb);
                }
            }
            b0 += nb;
        }
        if (!ok || *abort_flag) {
            if (leader) {
                atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
                *abort_flag = 1;
                tc_commit(drained);                                       // its products end before tensor memory is given back
                mbar_wait(drained, 0);
            }
            __syncwarp();
        }
    } else if (warp == PAGE_WARP) {
        // ---- the blocks' pages and exponents, ahead of the warps that convert them
        bool ok = true;
        int n = 0;                                                        // entries so far
        for (int round = 0; ok; round++) {
            const int item = item_of(round);
            const bool end = item >= n_items;
            Item t{};
            if (!end) t = load_item(p, list, item);
            int place = -1;                                               // this lane's page of 16 blocks, as its place in the pools
            for (int j = 0; j < (end ? 1 : t.nb) && ok; j++, n++) {
                if ((j & 15) == 0 && !end) {
                    const int page_idx = (t.blk0 + j) * 2 + lane;
                    place = -1;
                    if (page_idx <= t.key_hi / KV8_PAGE && page_idx >= t.key_lo / KV8_PAGE) {
                        const int page = p.block_table[(size_t)t.seq * p.table_stride + page_idx];
                        if (page >= 0 && page < p.n_pages) place = page * p.nkv + t.kvh;
                        else atomicOr(p.status, ESP_STATUS_BAD_INDEX);
                    }
                }
                const int mine = __shfl_sync(0xffffffffu, place, ((j & 15) * 2 + (lane >> 4)) & 31), s = n % AHEAD;
                uint2 e = make_uint2(0u, 0u);                             // 16 lanes a page, 8 exponents each
                if (!end && mine >= 0) e = *reinterpret_cast<const uint2*>(p.exps + (size_t)mine * 2 * KV8_PAGE + (lane & 15) * 8);
                ok = __all_sync(0xffffffffu, !*abort_flag && mbar_wait(&e_empty[s], ((n / AHEAD) & 1) ^ 1));
                if (!ok) break;
                Entry& x = entries[s];
                *reinterpret_cast<uint2*>(&x.exps[lane >> 4][0][0] + (lane & 15) * 8) = e;
                if ((lane & 15) == 0) x.block[lane >> 4] = mine;
                if (lane == 0) {
                    const int key0 = (t.blk0 + j) * BN;
                    x.lo = max(0, t.key_lo - key0);
                    x.hi = end ? -1 : min(BN, t.key_hi + 1 - key0);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&e_full[s]);
            }
            if (end) break;
        }
        if (!ok && lane == 0) {
            atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
            *abort_flag = 1;
        }
    } else if (warp >= MMA_WARP) {
        // no work: its registers went to the others
    } else if (warp >= ROW_WARPS) {
        // ---- codes to bfloat16.  A thread has a 16-channel piece c of R rows that follow one another (their exponents are one
        // load), and takes them in an order in which eight lanes' stores fall into different banks: half of the lanes
        // are at an odd row while the others are at an even one.  Keys and values of the blocks in turn; the codes of the next are
        // asked for when one has been converted, all together: a load asked for between two pieces would be waited for with
        // the next piece's, as a warp can tell only a few loads apart (418 cycles a piece).
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;\n");
        const int t = threadIdx.x - ROW_WARPS * 32;
        constexpr int R = HD == 128 ? 4 : 2;
        const int odd = (t >> 2) & 1, c = HD == 128 ? (t & 3) | ((t >> 1) & 4) : t & 3, row_lo = R * (HD == 128 ? (t >> 4) * 2 + odd : t >> 2);
        const bool whole_pieces = p.hd % 16 == 0;
        const bool live_lo = c * 16 < p.hd, live_hi = c * 16 + 8 < p.hd;  // the piece's halves that the heads have
        // row r of the piece goes to at ^ (r * 144) and its second half to that ^ 16: row r lies 128 r bytes further, its
        // 16-byte pieces swapped by r
        const unsigned to = (HD == 128 ? (c >> 2) * ATOM : 0) + row_lo * 128 + (((c & 3) * 2) << 4 ^ (row_lo & 7) << 4);
        const int half = row_lo / KV8_PAGE, in_page = row_lo % KV8_PAGE;
        // asks for a block's keys or values
        auto ask = [&](uint4 (&w)[R], const Entry& x, const unsigned char* pool) {
            const int block = x.block[half], a = x.lo - row_lo, b = x.hi - row_lo;
            const unsigned char* from = pool + ((size_t)max(block, 0) * KV8_PAGE + in_page) * p.hd + c * 16;
            if (block >= 0 && a <= 0 && b >= R && p.hd == HD) {
#pragma unroll
                for (int i = 0; i < R; i++) w[i] = *reinterpret_cast<const uint4*>(from + (i ^ odd) * HD);
            } else {
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const int r = i ^ odd;
                    const bool there = block >= 0 && r >= a && r < b;
                    w[i] = make_uint4(0u, 0u, 0u, 0u);
                    if (whole_pieces) {
                        if (there && live_lo) w[i] = *reinterpret_cast<const uint4*>(from + r * p.hd);
                    } else {
                        uint2 y = make_uint2(0u, 0u), z = y;
                        if (there && live_lo) y = *reinterpret_cast<const uint2*>(from + r * p.hd);
                        if (there && live_hi) z = *reinterpret_cast<const uint2*>(from + r * p.hd + 8);
                        w[i] = make_uint4(y.x, y.y, z.x, z.y);
                    }
                }
            }
        };
        // the codes times their powers of two, to the stage at ``at``
        auto convert = [&](const uint4 (&codes)[R], const Entry& x, const bool is_v, unsigned at) {
            typedef typename Word<R>::type Exps;                          // a byte for each of the thread's rows
            const unsigned ke = *reinterpret_cast<const Exps*>(&x.exps[half][0][in_page]), ve = *reinterpret_cast<const Exps*>(&x.exps[half][1][in_page]);
            // else: a position that is no number, or 2^(120 + e) beyond a bfloat16
            const bool plain = !__vcmpgtu4(ke, 0x86868686u) && !__vcmpgtu4(ve, 0x86868686u);
            if (__all_sync(0xffffffffu, plain)) {
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const unsigned word = is_v ? ve : ke;
                    // the byte of row i ^ odd, and 2^(120 + e) twice (of values 2^(120 - V_DOWN + e))
                    const unsigned f = ((odd ? word >> (8 * (i ^ 1)) : word >> (8 * i)) & 255u) * 0x00800080u + (120u - (is_v ? V_DOWN : 0)) * 0x00800080u;
                    const unsigned w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
                    unsigned o[8];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        o[2 * u] = mul_bf16x2(spread_codes<0x9180>(w[u]), f);
                        o[2 * u + 1] = mul_bf16x2(spread_codes<0xB3A2>(w[u]), f);
                    }
                    const unsigned dst = at ^ (unsigned)((i ^ odd) * 144);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst ^ 16u), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
                }
            } else {
#pragma unroll
                for (int i = 0; i < R; i++) {
                    const int r = i ^ odd;
                    const unsigned k8 = ke >> (8 * r) & 255u, v8 = ve >> (8 * r) & 255u;
                    const bool bad = (k8 == KV8_NAN || v8 == KV8_NAN) && r >= x.lo - row_lo && r < x.hi - row_lo;
                    const int up = (int)(is_v ? v8 : k8) + 120 - (is_v ? V_DOWN : 0), more = max(up - 254, 0);   // two factors
                    unsigned f = (unsigned)(up - more) << 7, f2 = (unsigned)(127 + more) << 7;
                    f = bad ? (is_v ? 0u : 0x7fffu) : f;                  // a key of NaN with a value of zeros
                    f2 = bad ? 0x3f80u : f2;
                    f |= f << 16;
                    f2 |= f2 << 16;
                    const unsigned w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
                    unsigned o[8];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        o[2 * u] = mul_bf16x2(mul_bf16x2(spread_codes<0x9180>(w[u]), f), f2);
                        o[2 * u + 1] = mul_bf16x2(mul_bf16x2(spread_codes<0xB3A2>(w[u]), f), f2);
                    }
                    const unsigned dst = at ^ (unsigned)(r * 144);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst ^ 16u), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7]) : "memory");
                }
            }
        };
        auto wait_all = [&](unsigned long long* bar, int parity) { return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity)); };
        // A block's keys are asked for behind the conversion of the values before them, and only then is it said that those are there.
        // (No load is on its way at the loop's end: there a warp would wait for it, 1,000 cycles a block.)
        uint4 codes[R];
        bool ok = true;
        auto values_done = [&](int n) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&v_full[n % STAGES]);
                mbar_arrive(&e_empty[n % AHEAD]);
            }
        };
        for (int n = 0;; n++) {
            ok = wait_all(&e_full[n % AHEAD], (n / AHEAD) & 1);
            if (!ok) break;
            const Entry& x = entries[n % AHEAD];
            const bool end = x.hi < 0;
            if (!end) ask(codes, x, p.k);
            if (n > 0) values_done(n - 1);
            if (end) break;
            const int st = n % STAGES, free_parity = ((n / STAGES) & 1) ^ 1;
            ok = wait_all(&k_empty[st], free_parity);
            if (!ok) break;
            convert(codes, x, false, smem_u32(k_s) + st * TILE + to);
            ask(codes, x, p.v);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&k_full[st]);
            ok = wait_all(&v_empty[st], free_parity);
            if (!ok) break;
            convert(codes, x, true, smem_u32(v_s) + st * TILE + to);
        }
        if (!ok && lane == 0) {
            atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
            *abort_flag = 1;
        }
    } else {
        // ---- row threads: TMEM lane = query row; two threads a row, each with 64 keys of a block
        asm volatile("setmaxnreg.inc.sync.aligned.u32 80;\n");
        const int quad = warp & 3, side = (warp >> 2) & 1, grp = warp >> 3, r = quad * 32 + lane;
        const unsigned lane_sel = (unsigned)(quad * 32) << 16;
        const int bar_grp = 1 + grp * 4 + quad, bar_row = 9 + quad;
        const float sc = p.scale_log2;
        const unsigned s_addr = tm_s + grp * BN + lane_sel + side * 64;
        const unsigned o_addr = tm_o + grp * BN + lane_sel;
        unsigned n_b = 0, ph_o = 0;                                       // blocks so far; a bit a group: the phase of its O
        float m_ref, l_run;                                              // the maximum that O and l_run are scaled by
        Item t;
        auto open = [&](int round) {
            const int item = item_of(round);
            if (item < n_items) t = load_item(p, list, item);
            return item < n_items;
        };
        auto two_tiles = [&]() { return t.pair; };
        auto meet = [&](bool across, bool ok) { return across ? all_agree(ok, bar_row, 128) : all_agree(ok, bar_grp, 64); };
        auto work = [&]() {
            bool ok = true;
            const int first_pos = t.pos0(grp), pos = first_pos + r;
            const int key_first = p.window > 0 ? pos - p.window + 1 : 0;             // may lie before the sequence's start
            int key_first_last = p.window > 0 ? max(0, first_pos + BM - p.window) : 0;   // of the tile's last row
            const int j0 = t.pair ? t.lo(grp, p.window) : grp, j1 = t.pair ? t.hi(grp) : t.nb - 1, step = t.pair ? 1 : 2;
            m_ref = -INFINITY, l_run = 0.f;
            // a page that is none among those of the item's keys (looked for while the first scores are on their way): all blocks are
            // treated as those at an edge
            if (misses_page(p.block_table, p.table_stride, p.n_pages, t.seq, t.key_lo, t.key_hi, lane)) key_first_last = INT_MAX;
            for (int j = j0; j <= j1; j += step, n_b++) {
                const int key0 = (t.blk0 + j) * BN;
                ok = mbar_wait(&s_full[grp], n_b & 1);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
                // live columns of an edge block: c_lo .. c_lo + c_span, one unsigned comparison each
                const bool edge = key0 + BN - 1 > first_pos || key0 < key_first_last;
                const int c_lo = key_first - key0 - side * 64;
                const unsigned c_span = (unsigned)(pos - key_first);
                // 32 scores at a time (all 64 in registers would spill, and what shared memory leaves of L1 does not hold spills), each read
                // once: their weights are taken by the maximum in use, ``ref``, unless they have outgrown it by 2^LAZY.  The row's threads
                // meet when their weights are written: seldom has one of them gone over to another maximum, and then both scale what
                // they have written, and O, to the larger one.  (A row's maxima are whole numbers, so that
                // scaling a weight is exact.)
                unsigned s[32];
                auto scores = [&](int at) {
                    tc_ask32(s_addr + at, s);
                    tc_wait_ld(s);
                    if (edge) {
                        // this thread's 64 keys are one page's: where it is none, no column
                        const bool none = key_first_last == INT_MAX && !has_page(p.block_table, p.table_stride, p.n_pages, t.seq, key0 + side * 64);
                        const int lo = none ? -1 : c_lo;
                        const unsigned span = none ? 0u : c_span;
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if ((unsigned)(at + i - lo) > span) s[i] = 0xff800000u;
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
#pragma unroll
                        for (int u = 0; u < 4; u++) m4[u] = fmaxf(fmaxf(m4[u], __uint_as_float(s[i + u])), __uint_as_float(s[i + u + 4]));
                    return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc;
                };
                float ref = m_ref, l_blk = 0.f;
                auto scale_weights = [&](unsigned at, int columns, float f) {
                    __nv_bfloat162 f2 = __float2bfloat162_rn(f);
                    tc_wait_st();
#pragma unroll 1
                    for (int u = 0; u < columns; u += 8) {
                        unsigned x[8];
                        tc_ld8(at + u, x);
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = mul_bf16x2(x[i], *reinterpret_cast<const unsigned*>(&f2));
                        tc_st8(at + u, x);
                    }
                };
                if (ok) {
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const float mx = scores(half * 32);
                        const bool far = mx > ref + LAZY;
                        if (__any_sync(0xffffffffu, far)) {
                            const float now = !far ? ref : ceilf(mx), f = far ? fast_exp2(ref - now) : 1.f;      // ref = -inf gives 0
                            if (half == 1) scale_weights(s_addr, 16, f);
                            l_blk *= f;
                            ref = now;
                        }
                        // the weights of 32 keys into 16 columns, over scores that have been read: P of the first 64 keys lies in the columns
                        // 0-31 of S, that of the others in 64-95
                        const float m_use = ref == -INFINITY ? 0.f : ref;
                        unsigned long long l_pair = 0ull;
                        const unsigned long long sc2 = pair_of(sc, sc), m2 = pair_of(-m_use, -m_use);
                        unsigned packed[8];
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const float2 x = parts_of(fma_pair(pair_of(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), sc2, m2));
                            const float a = fast_exp2(x.x), b = fast_exp2(x.y);
                            l_pair = add_pair(l_pair, pair_of(a, b));
                            packed[(i >> 1) & 7] = pack_bf16(a, b);
                            if (i % 16 == 14) tc_st8(s_addr + half * 16 + (i / 16) * 8, packed);
                        }
                        const float2 l2 = parts_of(l_pair);
                        l_blk += l2.x + l2.y;
                    }
                }
                const bool same = !__any_sync(0xffffffffu, ref != m_ref);
                if (!all_agree(ok && same, bar_grp, 64)) {                           // the same for both of a row's threads
                    float* xp = xmax + (grp * 2 + (n_b & 1)) * 256;                  // by turns
                    xp[side * 128 + r] = ref;
                    ok = all_agree(ok, bar_grp, 64);                                 // ... which go on or leave together
                    if (!ok) break;
                    const float now = fmaxf(ref, xp[(side ^ 1) * 128 + r]);
                    const float f = ref < now ? fast_exp2(ref - now) : 1.f, alpha = m_ref < now ? fast_exp2(m_ref - now) : 1.f;
                    scale_weights(s_addr, 32, f);
                    l_blk *= f;
                    l_run *= alpha;
                    m_ref = now;
                    if (j != j0) {
#pragma unroll 1
                        for (int u = side * (HD / 2); u < (side + 1) * (HD / 2); u += 8) {
                            unsigned x[8];
                            tc_ld8(o_addr + u, x);
#pragma unroll
                            for (int i = 0; i < 8; i++) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
                            tc_st8(o_addr + u, x);
                        }
                    }
                }
                l_run += l_blk;
                tc_wait_st();
                tc_fence_before();                                                   // S has been read, P and O written
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[grp]);
            }
            // ---- the item's end: the sum of the row's threads; with one tile for both groups their results are joined
            xsum[(grp * 2 + side) * 128 + r] = l_run;
            if (side == 0) xref[grp * 128 + r] = m_ref;
            for (int g = 0; g < 2; g++)
                if ((t.pair ? g == grp : g < t.nb) && ok) ok = !*abort_flag && mbar_wait(&o_full[g], ph_o >> g & 1);
            ph_o ^= t.pair || t.nb > 1 ? 3u : 1u;
            return ok;
        };
        auto finish = [&]() {
            const bool both = !t.pair && t.nb > 1;
            tc_fence_after();
            // a group without a key for this row counts 0 (and a row that is no number stays one: 0 * NaN)
            const int g0 = t.pair ? grp : 0;
            const float m0 = t.pair ? m_ref : xref[r], m1 = both ? xref[128 + r] : -INFINITY, m_all = fmaxf(m0, m1);
            float f0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - m_all), f1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - m_all);
            float l = f0 * (xsum[g0 * 256 + r] + xsum[g0 * 256 + 128 + r]);
            if (both) l += f1 * (xsum[256 + r] + xsum[384 + r]);
            // a row of one key: the weight as it was rounded, so that the result is its value
            if (p.window == 1 || t.pos0(0) + (t.pair ? grp * BM : 0) + r == 0) l = __bfloat162float(__float2bfloat16_rn(l));
            float inv = 1.f / l;                                     // 0 where all scores are -inf (an infinite query): 0 * inf is NaN
            if (l == 0.f) {                                          // ... or where the row has no key: zeros
                const int pos = t.pos0(grp) + r;
                if (!has_pages(p.block_table, p.table_stride, p.n_pages, t.seq, first_visible_key(pos, p.window, 0), pos)) inv = 0.f;
            }
            // what this thread takes from tensor memory: 32 columns of its row at a time.  Four lanes then exchange their pieces of eight, so that
            // a store writes 64 bytes of each of eight rows (of 32 rows it would write 16: 5,000 cycles an item).
            const int cols = t.pair ? HD / 2 : 32, col0 = (t.pair ? side : grp * 2 + side) * cols;
            const unsigned from = t.pair ? o_addr : tm_o + lane_sel;
            const int row_g = t.pair ? grp * BM : 0, n_rows = t.rows(grp), piece = lane & 3;
            inv *= (float)(1 << V_DOWN);
            f0 *= inv, f1 *= inv;
#pragma unroll 1
            for (int col = col0; col < col0 + cols && col < HD; col += 32) {
                uint4 w[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    unsigned x[8];
                    tc_ld8(from + col + u * 8, x);
                    float o[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) o[i] = __uint_as_float(x[i]) * f0;
                    if (both) {
                        tc_ld8(tm_o + BN + lane_sel + col + u * 8, x);
#pragma unroll
                        for (int i = 0; i < 8; i++) o[i] += __uint_as_float(x[i]) * f1;
                    }
                    w[u] = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
                }
                // w[u] of the group's lane i becomes piece i of its row u
#pragma unroll
                for (int bit = 1; bit <= 2; bit *= 2)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        if (u & bit) continue;
                        const bool up = piece & bit;
                        uint4 give = up ? w[u] : w[u + bit];
                        give.x = __shfl_xor_sync(0xffffffffu, give.x, bit), give.y = __shfl_xor_sync(0xffffffffu, give.y, bit);
                        give.z = __shfl_xor_sync(0xffffffffu, give.z, bit), give.w = __shfl_xor_sync(0xffffffffu, give.w, bit);
                        if (up) w[u] = give;
                        else w[u + bit] = give;
                    }
                const int c = col + piece * 8, r0 = r - piece;
                bf16* to = p.out + ((size_t)(t.row0 + row_g + r0) * p.nh + t.h) * p.hd + c;
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (r0 + u < n_rows && c < p.hd) *reinterpret_cast<uint4*>(to + (size_t)u * p.nh * p.hd) = w[u];
            }
            tc_fence_before();
            // the sums and O's have been read
            if (t.pair) named_sync(bar_grp, 64);
            else named_sync(bar_row, 128);
            if (lane == 0 && (t.pair || grp < t.nb)) mbar_arrive(&o_free[grp]);
        };
        if (!kv8_walk_items(open, two_tiles, work, meet, finish) && lane == 0) {
            atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
            *abort_flag = 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512));
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the queries [rows, heads, hd] in boxes of 128 rows x 1 head x 64 channels, zeros outside
int make_query_map(CUtensorMap* map, const void* base, long long rows, int nh, int hd) {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) != cudaSuccess || qres != cudaDriverEntryPointSuccess)
            return (int)cudaErrorNotSupported;
        fn = reinterpret_cast<EncodeTiledFn>(ptr);
    }
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)nh, (cuuint64_t)rows}, strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)hd * nh * 2};
    const cuuint32_t box[3] = {64, 1, BM}, elem[3] = {1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <int HD> int launch(const CUtensorMap& map_q, Params p, int device, cudaStream_t stream) {
    constexpr int TILE = HD / 64 * ATOM;
    const size_t smem = 1024 + (size_t)(2 + 2 * STAGES) * TILE + 288 + (8 + 4 + 2) * 128 * 4 + AHEAD * sizeof(Entry) + LIST * 2;
    static bool raised[64] = {false};
    static int sm_count[64] = {0};
    if (!raised[device]) {
        cudaError_t e = cudaFuncSetAttribute(attn_prefill_kv8_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sm_count[device], cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return (int)e;
        raised[device] = true;
    }
    p.smem_bytes = (int)smem;
    // An item for each SM at most: singly.  Many: in pairs, and in all launches, as a tile is left to its neighbour, which another launch may
    // list.  Between the two the kernel looks at what the tiles see.  Tiles of sequences of few new tokens count although another kernel has
    // them: looking there as well gains nothing (2,048 tokens beside 100 of one, 28 heads on 4, 257 us and 259 with a look; 1,000 beside
    // 100 of one 233 and 231; 700 behind 4,953 beside 60 of four, 32 on 8, 215 and 216; 100 of 33 beside 60 of one 226 and 233).
    const long long all_items = (long long)p.n_tiles * p.nh;
    p.way = (short)(all_items <= sm_count[device] ? SINGLY : all_items >= 4LL * sm_count[device] || p.n_tiles > FEW ? IN_PAIRS : LOOK);
    for (int at = 0; at < p.n_tiles; at += LIST) {
        Params q = p;
        q.tile_seq += at, q.tile_first += at;
        q.n_tiles = p.n_tiles - at < LIST ? p.n_tiles - at : LIST;
        const long long items = (long long)q.n_tiles * p.nh;
        const unsigned grid = (unsigned)(items < sm_count[device] ? items : sm_count[device]);
        esp_launch_pdl(ESP_PDL_MANY_ROWS, attn_prefill_kv8_kernel<HD>, dim3(grid), dim3(THREADS), smem, stream, map_q, q);
        const int rc = esp_launch_status();
        if (rc) return rc;
    }
    return 0;
}
}  // namespace

// q and out [n_tokens, nh, hd] bfloat16; tile_seq / tile_first: all tiles of 128 new tokens (sequence, the tile's first token among
// the sequence's new ones, a multiple of 128), best listed with those that see the most keys first; of sequences with at least ``least``
// new tokens; hd a multiple of 8 up to 128.
ESP_API int esp_attn_prefill_kv8(const void* q, long long n_tokens, const void* k, const void* v, const void* exps, void* out, const int* tile_seq,
                                 const int* tile_first, const int* seq_start, const int* seq_past, const int* block_table, int n_seqs, int table_stride,
                                 int n_pages, int n_tiles, int nh, int nkv, int hd, int window, int least, int* status, cudaStream_t stream) {
    if (n_tiles <= 0 || n_tokens <= 0) return 0;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh > 65535 || hd <= 0 || hd % 8 || hd > 128 || window < 0 || table_stride >= (1 << 25) || (long long)n_tiles * nh > 0x7fffffffLL || n_tokens > 0x7fffffffLL || least < 0 || least > BM)
        return (int)cudaErrorInvalidValue;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
    CUtensorMap map_q;
    const int rc = make_query_map(&map_q, q, n_tokens, nh, hd);
    if (rc) return rc;
    Params p{};
    p.k = (const unsigned char*)k, p.v = (const unsigned char*)v, p.exps = (const unsigned char*)exps, p.out = (bf16*)out;
    p.tile_seq = tile_seq, p.tile_first = tile_first, p.seq_start = seq_start, p.seq_past = seq_past, p.block_table = block_table, p.n_seqs = n_seqs;
    p.table_stride = table_stride, p.n_pages = n_pages, p.nh = nh, p.nkv = nkv, p.hd = hd, p.window = window, p.n_tiles = n_tiles, p.status = status;
    p.n_tokens = (int)n_tokens, p.least = (short)least;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
    if (hd <= 64) return launch<64>(map_q, p, device, stream);
    return launch<128>(map_q, p, device, stream);
}
