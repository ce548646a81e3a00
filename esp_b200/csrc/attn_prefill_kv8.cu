// Attention of many new tokens over the 8-bit paged cache (kv8.cuh) on the 5th-generation tensor cores: causal, optionally
// windowed, grouped query heads, runs of unequal length packed back to back.  Heads of up to 128 channels.
//
//   S = Q K^T      tcgen05.mma, 128 queries by 128 keys, accumulated in 32-bit in tensor memory
//   P = 2^(S log2(e) / sqrt(hd) - m)   in 32-bit, by the thread that owns the row; rounded to bfloat16 and written over S, where the next
//                  product reads it as its A operand
//   O += P V       tcgen05.mma, accumulated in tensor memory
//
// m is the row's running maximum, allowed to lag by 2^LAZY: O and the row's sum are rescaled only when it has outgrown that.
//
// The cache's codes cannot be operands beside bfloat16 queries and weights, so four warps turn them into bfloat16 on their way
// from global to shared memory: a code's bits moved into a bfloat16's places are the code times 2^-120, subnormal codes
// included, and one multiplication by 2^(120 + e) gives the number exactly.  That is four operations for two codes,
// 2.4 with loads and stores for each, against about 3.5 of the row threads for each score.  A block of keys is therefore made
// once for 256 queries: an item is two tiles of 128 new tokens of a sequence (PAIR), each with a group of row threads and S and O
// of its own, in all 512 columns of tensor memory.  Where there are few items, or a tile has no neighbour, the two groups
// take the blocks of one tile in turn instead (SPLIT) and join their results.
//
// A position that is no number (kv8.cuh) is made a key of NaN with a value of zeros: whoever sees it gets NaN through the score,
// and a masked score takes nothing of it.  Every wait is bounded.
#include "kv8.cuh"
#include "tc05.cuh"

namespace {
using namespace tc05;
constexpr int BM = 128, BN = 128, ATOM = 128 * 128;     // ATOM: bytes of a 64-channel slice of 128 rows
constexpr int STAGES = 2;                               // blocks of keys (and of values) in shared memory as bfloat16
// warps: 0-3 and 4-7 the groups of row threads, 8-11 codes to bfloat16, 12 MMA, 13 queries, 14 and 15 none.  Registers are moved
// between them (whole groups of four warps): 256 * 176 + 128 * 96 + 128 * 64 = 65,536, the launch's 512 * 128.
constexpr int ROW_WARPS = 8, CONV_WARPS = 4, MMA_WARP = 12, Q_WARP = 13, THREADS = 512;
constexpr int LIST = 4096;                              // tiles of a launch
constexpr float LAZY = 8.f;

struct Params {
    const unsigned char *k, *v, *exps;
    bf16* out;
    const int *tile_seq, *tile_first, *seq_start, *seq_past, *block_table;
    int table_stride, n_pages, nh, nkv, hd, window, n_tiles, pair, smem_bytes;
    float scale_log2;
    int* status;
};

__device__ __forceinline__ unsigned idesc_attn(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? (1u << 16) : 0u) | ((unsigned)(n >> 3) << 17) | ((unsigned)(128 >> 4) << 24);
}
// an MN-major operand: rows are consecutive keys, 128 bytes of channels each; the next 64 channels lie ``lbo`` bytes further
__device__ __forceinline__ unsigned long long smem_desc_mn(const void* p, unsigned lbo) {
    unsigned long long d = 0;
    d |= (unsigned long long)((smem_u32(p) & 0x3FFFFu) >> 4);
    d |= (unsigned long long)((lbo >> 4) & 0x3FFFu) << 16;
    d |= (unsigned long long)(1024 >> 4) << 32;
    d |= (unsigned long long)1 << 46;
    d |= (unsigned long long)2 << 61;
    return d;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
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
// the loads have arrived: their registers pass through here, so that no use is moved ahead of the wait
__device__ __forceinline__ void tc_wait_ld(unsigned (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
          "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
          "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]),
          "+r"(r[31])::"memory");
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
    const int tile = list[item / p.nh];
    t.h = item % p.nh;
    t.kvh = t.h / (p.nh / p.nkv);
    t.seq = p.tile_seq[tile];
    const int start = p.seq_start[t.seq];
    t.first = p.tile_first[tile];
    t.news = p.seq_start[t.seq + 1] - start;
    t.past = p.seq_past[t.seq];
    t.row0 = start + t.first;
    t.pair = p.pair && t.first + BM < t.news;
    t.key_lo = first_visible_key(t.pos0(0), p.window, 0);
    t.key_hi = t.pos0(1) + t.rows(1) - 1;
    t.blk0 = t.key_lo / BN;
    t.nb = t.key_hi / BN - t.blk0 + 1;
    return t;
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
                       *o_free = bars + 10, *k_full = bars + 12, *k_empty = k_full + STAGES, *v_full = k_empty + STAGES, *v_empty = v_full + STAGES;
    constexpr int N_BARS = 12 + 4 * STAGES;
    unsigned* tmem_slot = reinterpret_cast<unsigned*>(bars + N_BARS);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* n_active = reinterpret_cast<int*>(tmem_slot + 2);
    float* xsum = reinterpret_cast<float*>(bars + 32);   // [group][row]: the groups' sums where they share a tile
    float* xref = xsum + 2 * 128;                        // [group][row]: the maxima that they go with
    unsigned short* list = reinterpret_cast<unsigned short*>(xref + 2 * 128);
    static_assert(N_BARS <= 30, "the barriers and three words take 256 bytes");
    if (reinterpret_cast<unsigned char*>(list + LIST) > smem_raw + p.smem_bytes) {
        if (threadIdx.x == 0) atomicOr(p.status, ESP_STATUS_SMEM_LAYOUT);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < N_BARS; i++) mbar_init(&bars[i], 1);
        for (int g = 0; g < 2; g++) {
            mbar_init(&p_ready[g], 4);                   // a warp of the group's rows each
            mbar_init(&o_free[g], 4);
        }
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&k_full[s], CONV_WARPS);
            mbar_init(&v_full[s], CONV_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    pdl_wait();
    pdl_trigger();
    // ---- the tiles that begin an item, in the order of the list: with pairs, those whose place in their sequence is even
    if (warp == Q_WARP) {
        int n = 0;
        for (int i0 = 0; i0 < p.n_tiles; i0 += 32) {
            const int i = i0 + lane;
            const bool live = i < p.n_tiles && (!p.pair || (p.tile_first[i] / BM) % 2 == 0);
            const unsigned mask = __ballot_sync(0xffffffffu, live);
            if (live) list[n + __popc(mask & ((1u << lane) - 1u))] = (unsigned short)i;
            n += __popc(mask);
        }
        if (lane == 0) *n_active = n;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = *tmem_slot, tm_s = tmem, tm_o = tmem + 256;    // S of the groups at columns 0 and 128, O at 256 and 384
    const int n_items = *n_active * p.nh, G = gridDim.x;
    // block b takes the items b, 2G-1-b, 2G+b, ...: a long one is followed by a short one
    auto item_of = [&](int round) { return round * G + ((round & 1) ? G - 1 - (int)blockIdx.x : (int)blockIdx.x); };

    if (warp >= MMA_WARP) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
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
        if (lane == 0) {
            const unsigned idesc_s = idesc_attn(BN, false), idesc_pv = idesc_attn(HD, true);
            const unsigned long long dq = smem_desc(q_s), dk = smem_desc(k_s), dv = smem_desc_mn(v_s, ATOM);
            bool ok = true;
            int b0 = 0;                                                   // key blocks before this item
            unsigned ph_p = 0, ph_o = 0;                                  // a bit a group: the phase of its P, of its O
            for (int round = 0; ok && !*abort_flag; round++) {
                const int item = item_of(round);
                if (item >= n_items) break;
                const Item t = load_item(p, list, item);
                ok = mbar_wait(q_full, round & 1);
                tc_fence_after();
                unsigned begun = 0;                                       // a bit a group: its O holds something of this item
                auto issue_s = [&](int g, int j, bool last_use, bool last) {
                    const int st = (b0 + j) % STAGES;
                    if (!mbar_wait(&k_full[st], ((b0 + j) / STAGES) & 1)) return false;
                    tc_fence_after();
                    const unsigned long long a = dq + (t.pair ? (unsigned)(g * TILE) >> 4 : 0u), b = dk + ((st * TILE) >> 4);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const unsigned off = ((kk >> 2) * ATOM + (kk & 3) * 32) >> 4;
                        tc_mma(tm_s + g * BN, a + off, b + off, idesc_s, kk > 0 ? 1u : 0u);
                    }
                    tc_commit(&s_full[g]);
                    if (last_use) tc_commit(&k_empty[st]);
                    if (last) tc_commit(q_empty);
                    return true;
                };
                auto issue_pv = [&](int g, int j, bool last_use, bool last) {
                    const int st = (b0 + j) % STAGES;
                    // the row threads have read the O of the item before
                    if (!(begun >> g & 1) && !mbar_wait(&o_free[g], (ph_o >> g & 1) ^ 1)) return false;
                    if (!mbar_wait(&p_ready[g], ph_p >> g & 1) || !mbar_wait(&v_full[st], ((b0 + j) / STAGES) & 1)) return false;
                    tc_fence_after();
                    ph_p ^= 1u << g;
#pragma unroll
                    for (int kk = 0; kk < BN / 16; kk++)
                        tc_mma_ta(tm_o + g * BN, tm_s + g * BN + kk * 8, dv + ((st * TILE + kk * 16 * 128) >> 4), idesc_pv, kk > 0 ? 1u : begun >> g & 1);
                    if (!(begun >> g & 1)) ph_o ^= 1u << g;
                    begun |= 1u << g;
                    if (last_use) tc_commit(&v_empty[st]);
                    if (last) tc_commit(&o_full[g]);
                    return true;
                };
                // S of a block overwrites the P before it, so its group's P V comes first: the tensor core runs one
                // thread's products in the order in which they were issued
                if (t.pair) {
                    const int lo0 = t.lo(0, p.window), hi0 = t.hi(0), lo1 = t.lo(1, p.window), hi1 = t.hi(1);
                    for (int j = 0; j <= t.nb && ok && !*abort_flag; j++) {
                        if (ok && j - 1 >= lo0 && j - 1 <= hi0) ok = issue_pv(0, j - 1, j - 1 < lo1, j - 1 == hi0);
                        if (ok && j >= lo0 && j <= hi0) ok = issue_s(0, j, j < lo1, false);
                        if (ok && j - 1 >= lo1 && j - 1 <= hi1) ok = issue_pv(1, j - 1, true, j - 1 == hi1);
                        if (ok && j >= lo1 && j <= hi1) ok = issue_s(1, j, true, j == hi1);
                    }
                } else {
                    for (int j = 0; j < t.nb + 2 && ok && !*abort_flag; j++) {
                        if (j >= 2) ok = issue_pv(j & 1, j - 2, true, j >= t.nb);
                        if (ok && j < t.nb) ok = issue_s(j & 1, j, true, j + 1 == t.nb);
                    }
                }
                b0 += t.nb;
            }
            if (!ok) {
                atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
                *abort_flag = 1;
            }
            if (!ok || *abort_flag) {                                    // its products end before tensor memory is given back
                tc_commit(drained);
                mbar_wait(drained, 0);
            }
        }
    } else if (warp >= MMA_WARP) {
        // no work: two of the four warps whose registers went to the others
    } else if (warp >= ROW_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n");
        // ---- codes to bfloat16.  A thread has a 16-channel piece c of R rows that follow one another (their exponents are one
        // load), and takes them in an order in which eight lanes' stores fall into different banks: half of the lanes
        // are at an odd row while the others are at an even one.  Units of work, one behind the other: the keys of
        // block 0, then keys of block i and values of block i - 1 in turn.  A piece's registers get the next unit's codes as
        // soon as they have been converted.
        const int t = threadIdx.x - ROW_WARPS * 32;
        constexpr int R = HD == 128 ? 8 : 4;
        const int odd = (t >> 2) & 1, c = HD == 128 ? (t & 3) | ((t >> 1) & 4) : t & 3, row_lo = R * (HD == 128 ? (t >> 4) * 2 + odd : t >> 2);
        const bool whole_pieces = p.hd % 16 == 0;
        const int live_lo = c * 16 < p.hd, live_hi = c * 16 + 8 < p.hd;   // the piece's halves that the heads have
        struct Cursor {
            int round, u, seq, kvh, blk0, nb, key_lo, key_hi;
            bool done;
            __device__ __forceinline__ bool is_v() const { return u == 2 * nb - 1 || (u > 0 && (u & 1) == 0); }
            __device__ __forceinline__ int block() const { return u == 0 ? 0 : u == 2 * nb - 1 ? nb - 1 : (u & 1) ? (u + 1) / 2 : u / 2 - 1; }
        };
        auto open = [&](Cursor& cu, int round) {
            const int item = item_of(round);
            cu.done = item >= n_items;
            cu.round = round;
            cu.u = 0;
            if (cu.done) return;
            const Item it = load_item(p, list, item);
            cu.seq = it.seq, cu.kvh = it.kvh, cu.blk0 = it.blk0, cu.nb = it.nb, cu.key_lo = it.key_lo, cu.key_hi = it.key_hi;
        };
        auto next = [&](Cursor& cu) {
            if (!cu.done && ++cu.u == 2 * cu.nb) open(cu, cu.round + 1);
        };
        // this thread's page of a unit; -1: no rows of it are to be read
        auto page_of = [&](const Cursor& cu) {
            if (cu.done) return -1;
            const int key = (cu.blk0 + cu.block()) * BN + row_lo;
            if (key > cu.key_hi || key + R <= cu.key_lo) return -1;
            const int page = p.block_table[(size_t)cu.seq * p.table_stride + key / KV8_PAGE];
            if (page >= 0 && page < p.n_pages) return page;
            atomicOr(p.status, ESP_STATUS_BAD_INDEX);
            return -1;
        };
        struct Unit {                                                    // where a unit's rows are, and their exponents
            const unsigned char* src;
            unsigned rows;                                               // a bit for every row that is to be read
            unsigned long long ke, ve;
        };
        auto unit_of = [&](const Cursor& cu, int page) {
            Unit x{nullptr, 0u, 0ull, 0ull};
            if (page < 0) return x;
            const int key = (cu.blk0 + cu.block()) * BN + row_lo;
            const int a = max(0, cu.key_lo - key), b = min(R, cu.key_hi + 1 - key);
            x.rows = ((1u << b) - 1u) & ~((1u << a) - 1u);
            const size_t block = (size_t)page * p.nkv + cu.kvh;
            x.src = (cu.is_v() ? p.v : p.k) + (block * KV8_PAGE + key % KV8_PAGE) * p.hd + c * 16;
            const unsigned char* e = p.exps + block * 2 * KV8_PAGE + key % KV8_PAGE;
            if constexpr (R == 8) {
                x.ke = *reinterpret_cast<const unsigned long long*>(e);
                x.ve = *reinterpret_cast<const unsigned long long*>(e + KV8_PAGE);
            } else {
                x.ke = *reinterpret_cast<const unsigned*>(e);
                x.ve = *reinterpret_cast<const unsigned*>(e + KV8_PAGE);
            }
            return x;
        };
        auto read = [&](const Unit& x, int i) {
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            const int r = i ^ odd;
            if (x.rows >> r & 1) {
                const unsigned char* from = x.src + (size_t)r * p.hd;
                if (whole_pieces) {
                    if (live_lo) w = *reinterpret_cast<const uint4*>(from);
                } else {
                    if (live_lo) {
                        const uint2 y = *reinterpret_cast<const uint2*>(from);
                        w.x = y.x, w.y = y.y;
                    }
                    if (live_hi) {
                        const uint2 y = *reinterpret_cast<const uint2*>(from + 8);
                        w.z = y.x, w.w = y.y;
                    }
                }
            }
            return w;
        };
        Cursor cur, nxt;
        open(cur, 0);
        nxt = cur;
        next(nxt);
        Unit now = unit_of(cur, page_of(cur)), then;
        int page_then = page_of(nxt);
        uint4 buf[R];
#pragma unroll
        for (int i = 0; i < R; i++) buf[i] = read(now, i);
        int n_k = 0, n_v = 0;
        bool ok = true;
        while (!cur.done) {
            const bool is_v = cur.is_v();
            int& n = is_v ? n_v : n_k;
            const int st = n % STAGES;
            then = unit_of(nxt, page_then);
            ok = !*abort_flag && mbar_wait(is_v ? &v_empty[st] : &k_empty[st], ((n / STAGES) & 1) ^ 1);
            if (!__all_sync(0xffffffffu, ok)) {
                ok = false;
                break;
            }
            unsigned char* dst = (is_v ? v_s : k_s) + st * TILE + (HD == 128 ? (c >> 2) * ATOM : 0);
            const int piece = (c & 3) * 2;
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int r = i ^ odd, row = row_lo + r;
                const int ke = (int)(now.ke >> (8 * r)) & 255, ve = (int)(now.ve >> (8 * r)) & 255;
                const bool bad = (ke == KV8_NAN || ve == KV8_NAN) && (now.rows >> r & 1);
                const int byte = is_v ? ve : ke, up = byte + 120, more = max(up - 254, 0);
                // 2^(120 + e), in two factors where one bfloat16 does not hold it; a position that is no number: NaN, 0
                unsigned f = (unsigned)(up - more) << 7;
                f = bad ? (is_v ? 0u : 0x7fffu) : f;
                f |= f << 16;
                unsigned o[8];
                const unsigned w[4] = {buf[i].x, buf[i].y, buf[i].z, buf[i].w};
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    o[2 * u] = mul_bf16x2(spread_codes<0x9180>(w[u]), f);
                    o[2 * u + 1] = mul_bf16x2(spread_codes<0xB3A2>(w[u]), f);
                }
                if (more > 0 && !bad) {
                    const unsigned f2 = (unsigned)(127 + more) << 7, ff = f2 | f2 << 16;
#pragma unroll
                    for (int u = 0; u < 8; u++) o[u] = mul_bf16x2(o[u], ff);
                }
                unsigned char* at = dst + row * 128;
                *reinterpret_cast<uint4*>(at + ((piece ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                *reinterpret_cast<uint4*>(at + (((piece + 1) ^ (row & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
                buf[i] = read(then, i);
            }
            n++;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(is_v ? &v_full[st] : &k_full[st]);
            cur = nxt;
            now = then;
            next(nxt);
            page_then = page_of(nxt);
        }
        if (!ok && lane == 0) {
            atomicOr(p.status, ESP_STATUS_WAIT_EXPIRED);
            *abort_flag = 1;
        }
    } else {
        // ---- row threads: TMEM lane = query row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;\n");
        const int quad = warp & 3, grp = warp >> 2, r = quad * 32 + lane;
        const unsigned lane_sel = (unsigned)(quad * 32) << 16;
        const float sc = p.scale_log2;
        const unsigned s_addr = tm_s + grp * BN + lane_sel, o_addr = tm_o + grp * BN + lane_sel;
        bool ok = true;
        unsigned n_b = 0, ph_o = 0;                                       // blocks so far; a bit a group: the phase of its O
        for (int round = 0; ok; round++) {
            const int item = item_of(round);
            if (item >= n_items) break;
            const Item t = load_item(p, list, item);
            const int first_pos = t.pos0(grp), pos = first_pos + r;
            const int key_first = p.window > 0 ? pos - p.window + 1 : 0;             // may lie before the sequence's start
            const int key_first_last = p.window > 0 ? max(0, first_pos + BM - p.window) : 0;   // of the tile's last row
            const int j0 = t.pair ? t.lo(grp, p.window) : grp, j1 = t.pair ? t.hi(grp) : t.nb - 1, step = t.pair ? 1 : 2;
            float m_ref = -INFINITY, l_run = 0.f;                                    // the maximum that O and l_run are scaled by
            for (int j = j0; j <= j1; j += step, n_b++) {
                const int key0 = (t.blk0 + j) * BN;
                ok = !*abort_flag && mbar_wait(&s_full[grp], n_b & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                unsigned s[4][32];
#pragma unroll
                for (int c = 0; c < 4; c++) tc_ask32(s_addr + c * 32, s[c]);
#pragma unroll
                for (int c = 0; c < 4; c++) tc_wait_ld(s[c]);
                if (key0 + BN - 1 > first_pos || key0 < key_first_last) {
                    // live columns: c_lo .. c_lo + c_span, one unsigned comparison each
                    const int c_lo = key_first - key0;
                    const unsigned c_span = (unsigned)(pos - key_first);
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int i = 0; i < 32; i++)
                            if ((unsigned)(c * 32 + i - c_lo) > c_span) s[c][i] = 0xff800000u;
                }
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 32; i += 2)
#pragma unroll
                    for (int c = 0; c < 4; c++) m4[c] = fmaxf(fmaxf(m4[c], __uint_as_float(s[c][i])), __uint_as_float(s[c][i + 1]));
                const float m_new = fmaxf(m_ref, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc);
                const bool grew = m_new > m_ref + LAZY;
                if (j == j0) {
                    m_ref = m_new;
                } else if (__any_sync(0xffffffffu, grew)) {
                    const float alpha = grew ? fast_exp2(m_ref - m_new) : 1.f;       // m_ref = -inf gives 0
                    if (grew) m_ref = m_new;
                    l_run *= alpha;
#pragma unroll 1
                    for (int u = 0; u < HD; u += 16) {
                        float x[16];
                        unsigned y[16];
                        tc_ld16(o_addr + u, x);
#pragma unroll
                        for (int i = 0; i < 16; i++) y[i] = __float_as_uint(x[i] * alpha);
                        tc_st16(o_addr + u, y);
                    }
                }
                const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
                float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    unsigned packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float a = fast_exp2(fmaf(__uint_as_float(s[c][i]), sc, -m_use)), b = fast_exp2(fmaf(__uint_as_float(s[c][i + 1]), sc, -m_use));
                        l4[i & 2] += a;
                        l4[(i & 2) + 1] += b;
                        __nv_bfloat162 w = __floats2bfloat162_rn(a, b);
                        packed[i >> 1] = *reinterpret_cast<unsigned*>(&w);
                    }
                    tc_st16(s_addr + c * 16, packed);
                }
                tc_wait_st();
                l_run += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                tc_fence_before();                                                   // S has been read, P and O written
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[grp]);
            }
            if (!ok) break;
            // ---- the item's end: with two tiles each group has its own, with one the two groups' results are joined
            const bool both = !t.pair && t.nb > 1;
            if (!t.pair) {
                xsum[grp * 128 + r] = l_run;
                xref[grp * 128 + r] = m_ref;
            }
            for (int g = 0; g < 2; g++)
                if ((t.pair ? g == grp : g < t.nb) && ok) ok = !*abort_flag && mbar_wait(&o_full[g], ph_o >> g & 1);
            ph_o ^= t.pair || t.nb > 1 ? 3u : 1u;
            ok = t.pair ? (bool)__all_sync(0xffffffffu, ok) : all_agree(ok, 1 + quad, 64);
            if (!ok) break;
            tc_fence_after();
            const bool live = r < t.rows(grp);
            bf16* orow = p.out + ((size_t)(t.row0 + (t.pair ? grp * BM : 0) + r) * p.nh + t.h) * p.hd;
            // a group without a key for this row counts 0 (and a row that is no number stays one: 0 * NaN)
            const float m0 = t.pair ? m_ref : xref[r], m1 = both ? xref[128 + r] : -INFINITY, m_all = fmaxf(m0, m1);
            const float f0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - m_all), f1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - m_all);
            float l = f0 * (t.pair ? l_run : xsum[r]);
            if (both) l += f1 * xsum[128 + r];
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int col0 = t.pair ? 0 : grp * (HD / 2), cols = t.pair ? HD : HD / 2;      // what this thread writes
            const unsigned from = t.pair ? o_addr : tm_o + lane_sel;
#pragma unroll 1
            for (int col = col0; col < col0 + cols; col += 16) {
                float o[16];
                tc_ld16(from + col, o);
                if (both) {
                    float o1[16];
                    tc_ld16(tm_o + BN + lane_sel + col, o1);
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] = o[i] * f0 + o1[i] * f1;
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) o[i] *= f0;
                }
#pragma unroll
                for (int i = 0; i < 16; i += 8) {
                    if (!live || col + i >= p.hd) break;
                    __nv_bfloat162 w[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) w[u] = __floats2bfloat162_rn(o[i + 2 * u] * inv, o[i + 2 * u + 1] * inv);
                    *reinterpret_cast<uint4*>(orow + col + i) = make_uint4(*reinterpret_cast<unsigned*>(&w[0]), *reinterpret_cast<unsigned*>(&w[1]),
                                                                           *reinterpret_cast<unsigned*>(&w[2]), *reinterpret_cast<unsigned*>(&w[3]));
                }
            }
            tc_fence_before();
            if (t.pair) __syncwarp();
            else named_sync(1 + quad, 64);                                           // both O's and the sums have been read
            if (lane == 0 && (t.pair || grp < t.nb)) mbar_arrive(&o_free[grp]);
        }
        if (!ok && lane == 0) {
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
    const size_t smem = 1024 + (size_t)(2 + 2 * STAGES) * TILE + 256 + 4 * 128 * 4 + LIST * 2;
    static bool raised[64] = {false};
    static int sm_count[64] = {0};
    if (!raised[device]) {
        cudaError_t e = cudaFuncSetAttribute(attn_prefill_kv8_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sm_count[device], cudaDevAttrMultiProcessorCount, device);
        if (e != cudaSuccess) return (int)e;
        raised[device] = true;
    }
    p.smem_bytes = (int)smem;
    for (int at = 0; at < p.n_tiles; at += LIST) {
        Params q = p;
        q.tile_seq += at, q.tile_first += at;
        q.n_tiles = p.n_tiles - at < LIST ? p.n_tiles - at : LIST;
        const long long items = (long long)q.n_tiles * p.nh;
        // pairs halve the conversions and the number of items: not where the device would not be filled by them
        q.pair = items >= 4LL * sm_count[device];
        const unsigned grid = (unsigned)(items < sm_count[device] ? items : sm_count[device]);
        esp_launch_pdl(ESP_PDL_MANY_ROWS, attn_prefill_kv8_kernel<HD>, dim3(grid), dim3(THREADS), smem, stream, map_q, q);
        const int rc = esp_launch_status();
        if (rc) return rc;
    }
    return 0;
}
}  // namespace

// q and out [n_tokens, nh, hd] bfloat16; tile_seq / tile_first: all tiles of 128 new tokens (sequence, the tile's first token among
// the sequence's new ones), best listed with those that see the most keys first; hd a multiple of 8 up to 128.
ESP_API int esp_attn_prefill_kv8(const void* q, long long n_tokens, const void* k, const void* v, const void* exps, void* out, const int* tile_seq,
                                 const int* tile_first, const int* seq_start, const int* seq_past, const int* block_table, int table_stride,
                                 int n_pages, int n_tiles, int nh, int nkv, int hd, int window, int* status, cudaStream_t stream) {
    if (n_tiles <= 0 || n_tokens <= 0) return 0;
    if (nkv <= 0 || nh <= 0 || nh % nkv || nh > 65535 || hd <= 0 || hd % 8 || hd > 128 || window < 0 || (long long)n_tiles * nh > 0x7fffffffLL)
        return (int)cudaErrorInvalidValue;
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
    CUtensorMap map_q;
    const int rc = make_query_map(&map_q, q, n_tokens, nh, hd);
    if (rc) return rc;
    Params p{};
    p.k = (const unsigned char*)k, p.v = (const unsigned char*)v, p.exps = (const unsigned char*)exps, p.out = (bf16*)out;
    p.tile_seq = tile_seq, p.tile_first = tile_first, p.seq_start = seq_start, p.seq_past = seq_past, p.block_table = block_table;
    p.table_stride = table_stride, p.n_pages = n_pages, p.nh = nh, p.nkv = nkv, p.hd = hd, p.window = window, p.n_tiles = n_tiles, p.status = status;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
    if (hd <= 64) return launch<64>(map_q, p, device, stream);
    return launch<128>(map_q, p, device, stream);
}
