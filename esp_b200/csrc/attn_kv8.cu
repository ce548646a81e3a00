// Attention over the 8-bit paged cache (kv8.cuh), streaming: one new token of every sequence (decode), or sixteen new tokens of a
// run (head sizes that the tensor-memory kernel does not take, and sequences of few new tokens).
//
//   s_j = q k_j / sqrt(hd),  o = sum_j 2^(s_j log2 e - m) v_j / sum_j 2^(s_j log2 e - m),  m = max_j s_j log2 e
// over the keys max(0, pos - window + 1) <= j <= pos.
//
// A block has four warps and up to 8 * NT rows: the query heads that share one key/value head (decode), or consecutive
// tokens of one head (run).  Keys go by in units of 128, a chunk of 32 to each warp, which brings the codes of its chunks in by
// asynchronous copies (a ring of STAGES chunks, 16 bytes a lane, swizzled so that eight rows of an ldmatrix fall into
// different banks) and keeps a softmax and an output of its own; the warps' results are joined in ascending order.
//
// Decode is one stream: the units of all (row, key head) pairs, one behind the other, are dealt out evenly over a grid that the
// device holds at once, so that ragged lengths leave no block idle, and a block's copies run on across the pairs' borders.  A pair
// whose units fall to several blocks is put together by the last of them to finish, in the order of the blocks, so a result
// is the same in every run; how a row is divided depends on the lengths of the step's other rows.
//
// Both products run on mma.sync m16n8k16 in half precision with the cache as the 16-row operand, so a block of up to eight
// rows wastes no more than that: S^T = K Q^T, O^T = V^T P^T.  Codes become halfs exactly by one conversion per two codes
// (through bfloat16 it would be four operations), and the exponents are applied in 32-bit: a key's to its scores, a
// value's to its weight.  A half has little range, so
//   * queries are scaled by a power of two that brings the row's largest to 2^14 (bfloat16's 8 bits fit a half's 11),
//   * the weights 2^(s + e_v) have a running maximum M of their own, which may lag behind by 2^LAG_TOP; the largest weight lies
//     between 2^WEIGHT_TOP and 2^(WEIGHT_TOP + LAG_TOP), and what is below 2^-20 of it is rounded to multiples of 2^-30 of it.
// Sums, maxima and accumulators are 32-bit.  Weights and values far apart are held in this form; a warp leaves its result by the maximum of
// the scores alone, which may lag by 2^LAG_SUM, and moves that where large values' sums would pass 32-bit's range.
//
// Measured (B200, one launch behind another): 8 sequences of 4,096 keys, 16 heads of 128, 30.7 us for 135 MB; 64 ragged ones of
// up to 8,192, 28 heads on 4, 52 us for 231 MB; one of 131,071 34 us; one of 777 7.4 us.  The keys stream at the memory's rate
// (18 of the 30 us); of the rest a block's start takes 2.7 us (from the wait to its first chunk) and the joining of parts about 4 us
// a level (a fence, a count, two trips to L2); about 5 us are not accounted for, as every block has 13 or 14 units.  A grid of (row, head,
// split) blocks of one split length took 29.4, 86, 42.5 and 8.9 us, with the best length of each case 29.3, 60, 41 and 8.2.  Three blocks an
// SM with rings of two stages instead of two with three: 33.4, 53.7, 37.4 and 7.7 us.
// Heads are padded to 64, 96, 128, 192 or 256 channels (22 sequences of 7,411 keys, 5 heads of 80: 40.2 us in 96, 43.8 in 128; steps
// over channels that are not there left out at run time instead: 49, as the branches keep the loads of one step from the products of
// the last.  8 sequences of 4,096, 16 heads of 192: 43.7 us in 192, where two blocks fit an SM, 58 in 256).
#include "kv8.cuh"

namespace {
constexpr int THREADS = 128, WARPS = 4, CHUNK = 32, UNIT = WARPS * CHUNK, MAX_ROWS = 1024;
constexpr float WEIGHT_TOP = 6.f, LAG_TOP = 8.f, LAG_SUM = 40.f, RISE = 60.f;
// A value's exponent is added to its score, and above 2^24 a score has no place for it: scores whose maximum is this far from zero, or from the
// base they are counted from, are counted from that maximum.  (The place where that is looked for and done is seldom come to, but costs what it
// takes of registers and instructions: decode up to 1 %, sequences of few new tokens 2 %, prompts with wide heads more.  Scores counted from the row's maximum throughout,
// without a base: decode with sixteen rows a block 4 to 7 %, few new tokens 3 %.)
constexpr float FROM_ZERO = 1 << 20, FROM_BASE = 32.f;
constexpr int PARTS = 16;                      // of a pair, that one block joins

struct Params {
    const bf16* q;
    const unsigned char *k, *v, *exps;
    bf16* out;
    float* parts;                              // decode: [blocks][2][8 * NT][hd + 2] of the pairs that a block has a part of
    int* counters;                             // decode: per pair
    const int *tok_seq, *tok_pos;              // decode: per row of the step
    const int *seq_past, *seq_start;           // per sequence (decode: seq_past may be null)
    const int *tile_seq, *tile_first;          // run: tiles of 128 new tokens
    const int* block_table;
    int n_seqs, table_stride, n_pages, n_rows, nh, nkv, hd, window, most;      // n_seqs: rows of the page table; n_rows: of the queries; run, most: new tokens of the sequences it takes
    float scale_log2;                          // log2(e) / sqrt(hd)
    int* status;
};

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldsm_x4(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ unsigned transpose_8x8(unsigned a) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void mma_half(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned pack_half(float a, float b) {        // a in the low half
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ unsigned low_pair(unsigned r) { return kv8_half2((unsigned short)(r & 0xffffu)); }
__device__ __forceinline__ unsigned high_pair(unsigned r) { return kv8_half2((unsigned short)(r >> 16)); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
// copies ``bytes`` (0: fills with zeros) of a 16-byte, 8-byte, 4-byte piece
__device__ __forceinline__ void copy16(unsigned dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy8(unsigned dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

template <int HD> struct Ring {
    static constexpr int STAGES = HD == 64 ? 4 : HD >= 192 ? 2 : 3;
    static constexpr int ROW = HD == 96 ? 112 : HD == 192 ? 208 : HD;                      // bytes from row to row
    static constexpr int STAGE = CHUNK * ROW * 2 + 2 * CHUNK;            // keys, values, exponents of both
    static constexpr int WARP = (STAGES * STAGE + 127) / 128 * 128;
};
// where the 16-byte piece c of row r lies: rows of 64 bytes share 128 bytes with a neighbour; rows of 96 and 192 bytes lie 112 and 208
// apart, which keeps eight of them in different banks as they are
template <int HD> __device__ __forceinline__ int piece_at(int r, int c) {
    return Ring<HD>::ROW != HD ? r * Ring<HD>::ROW + (c << 4) : r * HD + ((c ^ (HD == 64 ? (r >> 1) & 3 : r & 7)) << 4);
}


// One warp's share: its ring of chunks, and the softmax and the output of the block's rows over the keys it has seen.
template <int HD, int NT, bool RUN> struct Stream {
    static constexpr int STAGES = Ring<HD>::STAGES, STAGE = Ring<HD>::STAGE, ROWS = 8 * NT, PP = HD / 16;
    unsigned qf[NT][HD / 16][2];
    float row_scale[NT][2];
    float o[NT][HD / 16][4], top[NT][2];       // top: M, of the row
    float m[NT][2], l[NT][2];                  // maximum (lagging by LAG_SUM) and sum of the lane's own keys
    float base[NT][2];                         // of the row: what its scores, m and top are counted from

    // asks for the chunk of keys key0 .. key0 + 31 in page ``page``; those outside [k0, k1] are filled with zeros
    static __device__ __forceinline__ void ask(const Params& p, unsigned char* st, int page, int kvh, int key0, int k0, int k1, int lane) {
        const unsigned k_dst = smem_addr(st), v_dst = k_dst + CHUNK * Ring<HD>::ROW, e_dst = v_dst + CHUNK * Ring<HD>::ROW;
        const bool wanted = key0 <= k1 && key0 + CHUNK > k0, ok = wanted && page >= 0 && page < p.n_pages;
        if (wanted && !ok && lane == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        const size_t block = ok ? (size_t)page * p.nkv + kvh : 0;
        const size_t row0 = (block * KV8_PAGE + key0 % KV8_PAGE) * p.hd;
        if (p.hd % 16 == 0) {
#pragma unroll
            for (int u = 0; u < PP; u++) {
                const int idx = u * 32 + lane, r = idx / PP, c = idx % PP;
                const bool live = ok && key0 + r >= k0 && key0 + r <= k1 && c * 16 < p.hd;
                const size_t from = row0 + (live ? (size_t)r * p.hd + c * 16 : 0);
                const int to = piece_at<HD>(r, c), bytes = live ? 16 : 0;
                copy16(k_dst + to, p.k + from, bytes);
                copy16(v_dst + to, p.v + from, bytes);
            }
        } else {
            for (int u = 0; u < 2 * PP; u++) {
                const int idx = u * 32 + lane, r = idx / (2 * PP), c = idx % (2 * PP);
                const bool live = ok && key0 + r >= k0 && key0 + r <= k1 && c * 8 < p.hd;
                const size_t from = row0 + (live ? (size_t)r * p.hd + c * 8 : 0);
                const int to = piece_at<HD>(r, c >> 1) + (c & 1) * 8, bytes = live ? 8 : 0;
                copy8(k_dst + to, p.k + from, bytes);
                copy8(v_dst + to, p.v + from, bytes);
            }
        }
        // the exponents: 32 bytes of the keys, 32 of the values (without a page: zeros, which hide its keys)
        if (lane < 16) copy4(e_dst + lane * 4, p.exps + (block * 2 + (lane >> 3)) * KV8_PAGE + key0 % KV8_PAGE + (lane & 7) * 4, ok ? 4 : 0);
    }

    // the rows' queries: row r at q + r * step, those from ``rows`` on zero
    static __device__ __forceinline__ void ask_queries(uint2 (&raw)[NT][HD / 16], const bf16* q, long long step, int rows, int hd, int lane) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 8 + (lane >> 2);
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                const int d = kk * 16 + (lane & 3) * 4;
                raw[nt][kk] = r < rows && d < hd ? *reinterpret_cast<const uint2*>(q + r * step + d) : make_uint2(0u, 0u);
            }
        }
    }
    // ... as B operands, scaled row by row; row_scale: what a score is multiplied by (before the key's exponent).  Empties the rest.
    __device__ __forceinline__ void begin(const uint2 (&raw)[NT][HD / 16], float scale_log2, int lane) {
        const int tg = lane & 3;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float amax = 0.f;
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[nt][kk].x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[nt][kk].y));
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int x = max((int)(__float_as_uint(amax) >> 23) - 127, -100);       // the largest lies in [2^x, 2^(x+1))
            const float f = x > 127 ? __int_as_float(0x7fffffff) : kv8_pow2(14 - x);    // an infinite query is no number: 0 / 0 or inf / inf
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[nt][kk].x)), b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[nt][kk].y));
                qf[nt][kk][0] = pack_half(a.x * f, a.y * f);
                qf[nt][kk][1] = pack_half(b.x * f, b.y * f);
            }
            // a lane's scores belong to rows 2 tg and 2 tg + 1, whose queries the lanes 8 tg and 8 tg + 4 hold
            const int xa = __shfl_sync(0xffffffffu, x, tg * 8), xb = __shfl_sync(0xffffffffu, x, tg * 8 + 4);
            // times 2^16, and a key's factor by 2^-16: neither product passes 32-bit's range unless the score does
            row_scale[nt][0] = kv8_pow2(min(xa - 14, 127)) * (scale_log2 * 65536.f);
            row_scale[nt][1] = kv8_pow2(min(xb - 14, 127)) * (scale_log2 * 65536.f);
#pragma unroll
            for (int i = 0; i < HD / 16; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[nt][i][j] = 0.f;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                m[nt][j] = top[nt][j] = -INFINITY;
                l[nt][j] = base[nt][j] = 0.f;
            }
        }
    }

    // Scores far from zero: counted from the rows' bases (as they are rounded: equal ones stay equal), which are moved to the rows' maxima where
    // those have gone away from them.
    __device__ __forceinline__ void rebase(int nt, float (&s)[NT][2][4], float (&t)[4][2], float (&cm)[2], float (&ct)[2], const float (&ve)[4]) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            cm[j] = ct[j] = -INFINITY;
#pragma unroll
            for (int u = 0; u < 4; u++) cm[j] = fmaxf(cm[j], s[nt][u >> 1][(u & 1) * 2 + j] -= base[nt][j]);
            float row = fmaxf(m[nt][j], cm[j]), d = 0.f;
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) row = fmaxf(row, __shfl_xor_sync(0xffffffffu, row, off));
            if (fabsf(row) > (base[nt][j] == 0.f ? FROM_ZERO : FROM_BASE) && fabsf(row) < INFINITY) {
                const float now = base[nt][j] + rintf(row);
                d = now - base[nt][j];
                base[nt][j] = now;
            }
            m[nt][j] -= d, top[nt][j] -= d, cm[j] -= d;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                t[u][j] = (s[nt][u >> 1][(u & 1) * 2 + j] -= d) + ve[u];
                ct[j] = fmaxf(ct[j], t[u][j]);
            }
        }
    }

    // the chunk of keys key0 .. key0 + 31 that lies in ``st``; [k0, k1]: the keys that the block's rows see (run: row r sees those up
    // to pos0 + r, and of them the last ``window``)
    __device__ __forceinline__ void chunk(const unsigned char* st, int key0, int k0, int k1, int pos0, int window, int lane) {
        const int g8 = lane >> 2, tg = lane & 3;
        const unsigned k_src = smem_addr(st), v_src = k_src + CHUNK * Ring<HD>::ROW;
        const unsigned char* e_src = st + 2 * CHUNK * Ring<HD>::ROW;
        // ---- S^T: 32 keys (two tiles of 16) by the rows
        float s[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[nt][mt][j] = 0.f;
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int kp = 0; kp < HD / 32; kp++) {
                // codes 4 tg .. 4 tg + 3 of the 16 channels: the first two are the operand's columns 2 tg, 2 tg + 1, the others
                // its columns 2 tg + 8, 2 tg + 9; the queries' fragments are laid out the same way
                unsigned r[4];
                ldsm_x4(r, k_src + piece_at<HD>(mt * 16 + (lane & 15), 2 * kp + (lane >> 4)));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const unsigned a0 = low_pair(r[2 * h]), a1 = low_pair(r[2 * h + 1]), a2 = high_pair(r[2 * h]), a3 = high_pair(r[2 * h + 1]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma_half(s[nt][mt], a0, a1, a2, a3, qf[nt][2 * kp + h][0], qf[nt][2 * kp + h][1]);
                }
            }
        // ---- scores in units of log2; this lane's keys are key0 + 8 u + g8, u = 0 .. 3
        float kf[4], ve[4];
        bool seen[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int key = key0 + u * 8 + g8, ke = e_src[u * 8 + g8], vb = e_src[CHUNK + u * 8 + g8];
            seen[u] = key >= k0 && key <= k1 && ke != 0;                  // a stored exponent is never 0: the page was not one
            kf[u] = ke == KV8_NAN || vb == KV8_NAN ? __int_as_float(0x7fffffff) : __uint_as_float((unsigned)(ke - 16) << 23);
            ve[u] = (float)(vb - 127);
        }
        unsigned wf[NT][4];                    // the weights as B operands: keys 8 u .. 8 u + 7 by rows
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float t[4][2], cm[2] = {-INFINITY, -INFINITY}, ct[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float x = s[nt][u >> 1][(u & 1) * 2 + j] * kf[u] * row_scale[nt][j];
                    bool live = seen[u];
                    if constexpr (RUN) {
                        const int key = key0 + u * 8 + g8, pos = pos0 + nt * 8 + 2 * tg + j;
                        live = live && key <= pos && (window <= 0 || pos - key < window);
                    }
                    if (!live) x = -INFINITY;
                    s[nt][u >> 1][(u & 1) * 2 + j] = x;
                    t[u][j] = x + ve[u];
                    cm[j] = fmaxf(cm[j], x);
                    ct[j] = fmaxf(ct[j], t[u][j]);
                }
            // what is in use has been outgrown: the first chunk, and seldom after it
            bool far = base[nt][0] != 0.f || base[nt][1] != 0.f;
            far = far || cm[0] > m[nt][0] + LAG_SUM || cm[1] > m[nt][1] + LAG_SUM || ct[0] > top[nt][0] + LAG_TOP || ct[1] > top[nt][1] + LAG_TOP;
            if (__any_sync(0xffffffffu, far)) {
                const float c0 = fabsf(fmaxf(m[nt][0], cm[0])), c1 = fabsf(fmaxf(m[nt][1], cm[1]));
                const bool large = base[nt][0] != 0.f || base[nt][1] != 0.f || (c0 > FROM_ZERO && c0 < INFINITY) || (c1 > FROM_ZERO && c1 < INFINITY);
                if (__any_sync(0xffffffffu, large)) rebase(nt, s, t, cm, ct, ve);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    cm[j] = fmaxf(m[nt][j], cm[j]);
                    if (cm[j] > m[nt][j]) l[nt][j] *= exp2_fast(m[nt][j] - cm[j]);
                    m[nt][j] = cm[j];
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) ct[j] = fmaxf(ct[j], __shfl_xor_sync(0xffffffffu, ct[j], off));
                    ct[j] = fmaxf(top[nt][j], ct[j]);
                    const float f = ct[j] > top[nt][j] ? exp2_fast(top[nt][j] - ct[j]) : 1.f;
                    top[nt][j] = ct[j];
#pragma unroll
                    for (int d = 0; d < HD / 16; d++) {
                        o[nt][d][j] *= f;
                        o[nt][d][j + 2] *= f;
                    }
                }
            }
            const float mu[2] = {m[nt][0] == -INFINITY ? 0.f : m[nt][0], m[nt][1] == -INFINITY ? 0.f : m[nt][1]};
            const float tu[2] = {(top[nt][0] == -INFINITY ? 0.f : top[nt][0]) - WEIGHT_TOP, (top[nt][1] == -INFINITY ? 0.f : top[nt][1]) - WEIGHT_TOP};
#pragma unroll
            for (int u = 0; u < 4; u++) {
#pragma unroll
                for (int j = 0; j < 2; j++) l[nt][j] += exp2_fast(s[nt][u >> 1][(u & 1) * 2 + j] - mu[j]);
                wf[nt][u] = transpose_8x8(pack_half(exp2_fast(t[u][0] - tu[0]), exp2_fast(t[u][1] - tu[1])));
            }
        }
        // ---- O^T += V^T P^T: row r < 8 of an operand tile is channel 2 r of its 16, row r + 8 channel 2 r + 1
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            unsigned r[4];
            ldsm_x4_trans(r, v_src + piece_at<HD>(lane, d));
#pragma unroll
            for (int u = 0; u < 4; u++) r[u] = __byte_perm(r[u], 0, 0x3120);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const unsigned a0 = low_pair(r[2 * h]), a1 = high_pair(r[2 * h]), a2 = low_pair(r[2 * h + 1]), a3 = high_pair(r[2 * h + 1]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma_half(o[nt][d], a0, a1, a2, a3, wf[nt][2 * h], wf[nt][2 * h + 1]);
            }
        }
    }

    // the result in the form (m, l, sum of weights 2^(s - m) times values): m and l of the rows to the lists, the sum to o_w [ROWS][HD]
    __device__ __forceinline__ void leave(float* m_w, float* l_w, float* o_w, int lane) {
        const int g8 = lane >> 2, tg = lane & 3;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float most = m[nt][j];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, off));
                // by the base itself where there is one, as a large base plus a small number is not exact
                if (base[nt][j] != 0.f) most = 0.f;
                // a lane without a key counts 0; one whose keys are no numbers is NaN and stays it
                float sum = l[nt][j] * (m[nt][j] == -INFINITY ? 0.f : exp2_fast(m[nt][j] - most));
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                // values of large exponents above a maximum that lags: the sums of weights times values would pass 32-bit's range, so
                // the maximum is moved to where the sum of the weights is between 1 and 2.  (Up to 2^RISE they are in it: o stays below
                // 2^14 * 448 * 2^24 keys.)
                if (most > -INFINITY && top[nt][j] - WEIGHT_TOP - most > RISE && sum < INFINITY) {
                    const int up = max((int)(__float_as_uint(sum) >> 23) - 127, 0);
                    most += (float)up;
                    sum *= kv8_pow2(-up);
                }
                const int r = nt * 8 + 2 * tg + j;
                const float f = most == -INFINITY ? 1.f : exp2_fast(top[nt][j] - WEIGHT_TOP - most);
                if (g8 == 0) {
                    m_w[r] = base[nt][j] + most;
                    l_w[r] = sum;
                }
#pragma unroll
                for (int d = 0; d < HD / 16; d++)
                    *reinterpret_cast<float2*>(o_w + r * HD + d * 16 + 2 * g8) = make_float2(o[nt][d][j] * f, o[nt][d][j + 2] * f);
            }
    }
};

// The warps' results of row r, channels d and d + 1, in ascending order of the warps: (maximum, sum, the two sums of values).  A warp
// that saw nothing has m = -inf, l = 0, o = 0; one that saw only positions that are not numbers has m = -inf and NaN in l
// and o, which stay (0 * NaN = NaN).  ``o_s``: the first warp's sums, the others' ``warp_bytes`` behind one another.
struct Joined {
    float m, l, a, b;
};
template <int ROWS, int HD>
__device__ __forceinline__ Joined join_warps(const float (*m_s)[ROWS], const float (*l_s)[ROWS], const unsigned char* o_s, int warp_bytes, int r, int d) {
    Joined x{-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < WARPS; u++) x.m = fmaxf(x.m, m_s[u][r]);
#pragma unroll
    for (int u = 0; u < WARPS; u++) {
        const float w = m_s[u][r] == -INFINITY ? 0.f : exp2_fast(m_s[u][r] - x.m);
        const float2 v = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(o_s + u * warp_bytes) + r * HD + d);
        x.l += l_s[u][r] * w;
        x.a += v.x * w;
        x.b += v.y * w;
    }
    return x;
}
// the sum is 0 where none of the row's pages was one
__device__ __forceinline__ float inverse(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }
__device__ __forceinline__ void store_pair(bf16* to, float a, float b) { *reinterpret_cast<__nv_bfloat162*>(to) = __floats2bfloat162_rn(a, b); }

// ---------------------------------------------------------------------------------------------------- sixteen tokens of a run
// Bound by its instructions: every block of sixteen tokens converts the keys that they see.  2,048 tokens: 16 heads of 192 250 us (two
// blocks an SM; padded to 256 channels, one block, 400), 8 of 256 240 us, 103 and 72 TFLOP/s.
template <int HD, int NT>
__global__ void __launch_bounds__(THREADS) attn_run_kv8_kernel(const Params p) {
    pdl_trigger();
    typedef Stream<HD, NT, true> S;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float m_s[WARPS][S::ROWS], l_s[WARPS][S::ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* ring = smem + warp * Ring<HD>::WARP;
    pdl_wait();
    // the block's rows: ``rows`` tokens from ``first`` on, all of head ``head``
    const int subs = 128 / S::ROWS, tile = blockIdx.x / subs, seq = p.tile_seq[tile], tile_first = p.tile_first[tile], first = tile_first + (blockIdx.x % subs) * S::ROWS;
    if (seq < 0 || seq >= p.n_seqs || tile_first < 0 || tile_first % 128) {
        if (threadIdx.x == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        return;
    }
    const int start = p.seq_start[seq], end = p.seq_start[seq + 1], head = blockIdx.y, kvh = head / (p.nh / p.nkv);
    // rows that the queries do not have are looked for first: only where there are none is end - start a number of rows
    const bool there = (unsigned)start <= (unsigned)end && (unsigned)end <= (unsigned)p.n_rows;
    const int rows = there ? min(S::ROWS, end - start - first) : 0;
    if (rows <= 0) {                           // or behind the sequence's last token; a whole tile there is none
        if (threadIdx.x == 0 && first == tile_first) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        return;
    }
    const int past = p.seq_past[seq];
    if (past < 0 || ((long long)past + first + rows - 1) / KV8_PAGE >= p.table_stride) {           // positions that the page table does not have
        if (threadIdx.x == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        return;
    }
    if (end - start > p.most) return;          // the tensor-memory kernel's
    const int pos0 = past + first, k0 = first_visible_key(pos0, p.window, 0), k1 = pos0 + rows - 1;
    const long long row0 = (long long)(start + first) * p.nh + head;
    const int n_chunks = k1 / CHUNK - k0 / CHUNK + 1, mine = (n_chunks - warp + WARPS - 1) / WARPS;
    const int* pages = p.block_table + (size_t)seq * p.table_stride;
    auto key_of = [&](int i) { return (k0 / CHUNK + i * WARPS + warp) * CHUNK; };
    auto page_of = [&](int i) { return i < mine ? pages[key_of(i) / KV8_PAGE] : -1; };
    auto load = [&](int i, int page) {
        if (i < mine) S::ask(p, ring + (i % S::STAGES) * S::STAGE, page, kvh, key_of(i), k0, k1, lane);
        copies_commit();
    };
    int page_next = page_of(0);                // read one chunk ahead
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; s++) {
        const int page = page_next;
        page_next = page_of(s + 1);
        load(s, page);
    }
    S x;
    {
        uint2 raw[NT][HD / 16];
        S::ask_queries(raw, behind_wait(p.q) + row0 * p.hd, (long long)p.nh * p.hd, rows, p.hd, lane);
        x.begin(raw, p.scale_log2, lane);
    }
    for (int i = 0; i < mine; i++) {
        copies_wait<S::STAGES - 2>();
        __syncwarp();                          // every lane's pieces of chunk i are there, and all have read chunk i - 1
        const int page = page_next;
        page_next = page_of(i + S::STAGES);
        load(i + S::STAGES - 1, page);
        x.chunk(ring + (i % S::STAGES) * S::STAGE, key_of(i), k0, k1, pos0, p.window, lane);
    }
    copies_wait<0>();
    __syncwarp();
    x.leave(m_s[warp], l_s[warp], reinterpret_cast<float*>(ring), lane);
    __syncthreads();
    const int pairs = p.hd / 2;
    for (int idx = threadIdx.x; idx < rows * pairs; idx += THREADS) {
        const int r = idx / pairs, d = (idx % pairs) * 2;
        const Joined y = join_warps<S::ROWS, HD>(m_s, l_s, smem, Ring<HD>::WARP, r, d);
        store_pair(p.out + (row0 + (long long)r * p.nh) * p.hd + d, y.a * inverse(y.l), y.b * inverse(y.l));
    }
}

// ---------------------------------------------------------------------------------------------------- one token of every sequence
// What a unit of the stream belongs to.
struct Cursor {
    int row, kvb, unit, last;                  // the step's row, its block of heads, the unit's place among absolute 128 keys; the pair's last
    int seq, pos, lo;                          // of the row; pos < 0: no row
};

template <int HD, int NT>
__global__ void __launch_bounds__(THREADS) attn_decode_kv8_kernel(const Params p) {
    pdl_trigger();
    typedef Stream<HD, NT, false> S;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float m_s[WARPS][S::ROWS], l_s[WARPS][S::ROWS];
    __shared__ int before[MAX_ROWS + 1];       // units of one key head ahead of each row
    __shared__ int warp_sum_s[WARPS], is_last;
    __shared__ float2 joined_ml[S::ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned char* ring = smem + warp * Ring<HD>::WARP;
    const int group = p.nh / p.nkv, per_kv = (group + S::ROWS - 1) / S::ROWS, kv_blocks = p.nkv * per_kv;

    // a row's units; one whose position is not in the table has none
    auto units_of = [&](int pos) {
        return pos < 0 || pos / KV8_PAGE >= p.table_stride ? 0 : pos / UNIT - first_visible_key(pos, p.window, 0) / UNIT + 1;
    };
    // ---- how many units lie ahead of each row (every block works it out for itself; rows and positions were there before this step's
    // kernels began)
    int carry = 0;
    for (int r0 = 0; r0 < p.n_rows; r0 += THREADS) {
        const int r = r0 + threadIdx.x;
        int mine = 0;
        if (r < p.n_rows) {
            const int pos = p.tok_pos[r];
            mine = p.tok_seq[r] < 0 || p.tok_seq[r] >= p.n_seqs ? 0 : units_of(pos);
            if (mine == 0 && blockIdx.x == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        }
        int sum = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, off);
            if (lane >= off) sum += v;
        }
        if (lane == 31) warp_sum_s[warp] = sum;
        __syncthreads();
        int ahead = carry, all = carry;
#pragma unroll
        for (int u = 0; u < WARPS; u++) {
            if (u < warp) ahead += warp_sum_s[u];
            all += warp_sum_s[u];
        }
        if (r < p.n_rows) before[r] = ahead + sum - mine;
        carry = all;
        __syncthreads();
    }
    if (threadIdx.x == 0) before[p.n_rows] = carry;
    __syncthreads();
    const long long total = (long long)carry * kv_blocks;
    const int blocks = (int)min((long long)gridDim.x, total);            // that have units: each of them one at least
    if ((int)blockIdx.x >= blocks) {
        pdl_wait();                            // a grid without units ends behind the kernel before it, too
        return;
    }
    const long long u0 = total * blockIdx.x / blocks, u1 = total * (blockIdx.x + 1) / blocks;

    // ---- cursors through the stream: pairs row by row, of a row its blocks of heads one behind the other
    auto open_row = [&](Cursor& c) {
        c.seq = p.tok_seq[c.row];
        c.pos = p.tok_pos[c.row];
        c.lo = first_visible_key(c.pos, p.window, 0);
        c.last = c.pos / UNIT;
    };
    auto advance = [&](Cursor& c) {
        if (c.unit < c.last) {
            c.unit++;
        } else if (c.kvb + 1 < kv_blocks) {
            c.kvb++;
            c.unit = c.lo / UNIT;
        } else {
            do c.row++;
            while (c.row < p.n_rows && before[c.row] == before[c.row + 1]);   // rows without units
            c.kvb = 0;
            if (c.row < p.n_rows) {
                open_row(c);
                c.unit = c.lo / UNIT;
            }
        }
    };
    Cursor now;
    {
        int a = 0, b = p.n_rows;               // the last row whose units begin at or ahead of u0, and that has some
        while (b - a > 1) {
            const int mid = (a + b) / 2;
            if ((long long)before[mid] * kv_blocks <= u0) a = mid;
            else b = mid;
        }
        now.row = a;
        open_row(now);
        const long long in_row = u0 - (long long)before[a] * kv_blocks;
        const int each = before[a + 1] - before[a];
        now.kvb = (int)(in_row / each);
        now.unit = now.lo / UNIT + (int)(in_row % each);
    }
    const int n_units = (int)(u1 - u0);
    Cursor ahead = now;                        // of the chunk behind the one that is asked for next
    int asked = 0;
    auto page_of = [&](const Cursor& c) { return p.block_table[(size_t)c.seq * p.table_stride + min(c.unit * UNIT + warp * CHUNK, c.pos) / KV8_PAGE]; };
    // the next chunk of this warp, into the ring's next stage
    auto load = [&](const Cursor& c, int page) {
        if (asked < n_units) S::ask(p, ring + (asked % S::STAGES) * S::STAGE, page, c.kvb / per_kv, c.unit * UNIT + warp * CHUNK, c.lo, c.pos, lane);
        asked++;
        copies_commit();
    };
    // the first chunks' pages are looked up at once, the later ones' one chunk ahead
    Cursor first[S::STAGES];
    int first_page[S::STAGES];
#pragma unroll
    for (int i = 0; i < S::STAGES; i++) {
        first[i] = ahead;
        first_page[i] = page_of(ahead);
        if (i + 1 < n_units) advance(ahead);
    }
    auto head_of = [&](const Cursor& c) { return c.kvb / per_kv * group + c.kvb % per_kv * S::ROWS; };
    auto rows_of = [&](const Cursor& c) { return min(S::ROWS, group - c.kvb % per_kv * S::ROWS); };
    // Positions that were cached before this step do not depend on the kernel before this one, which writes the step's own: where
    // the first chunks are older, they are asked for at once, and only then come the wait and the queries.
    const bool early = p.seq_past != nullptr && now.unit + S::STAGES - 2 <= now.last && min((now.unit + S::STAGES - 1) * UNIT - 1, now.pos) < p.seq_past[now.seq];
    uint2 raw[NT][HD / 16];
    const bf16* q;
    auto ask_first = [&]() {
        pdl_wait();
        q = behind_wait(p.q);
        S::ask_queries(raw, q + ((size_t)now.row * p.nh + head_of(now)) * p.hd, p.hd, rows_of(now), p.hd, lane);
    };
    if (!early) ask_first();
#pragma unroll
    for (int i = 0; i < S::STAGES - 1; i++) load(first[i], first_page[i]);
    if (early) ask_first();
    Cursor next = first[S::STAGES - 1];
    int page_next = first_page[S::STAGES - 1];

    const int pairs = p.hd / 2, part = S::ROWS * (p.hd + 2);             // floats of a part: the sums, then (m, l) of the rows
    S x;
    int began = now.unit;                      // the first of the pair's units that is this block's
    x.begin(raw, p.scale_log2, lane);
    for (int i = 0; i < n_units; i++) {
        copies_wait<S::STAGES - 2>();
        __syncwarp();                          // every lane's pieces of chunk i are there, and all have read chunk i - 1
        load(next, page_next);
        if (asked < n_units) {
            next = ahead;
            page_next = page_of(next);
            if (asked + 1 < n_units) advance(ahead);
        }
        unsigned char* st = ring + (i % S::STAGES) * S::STAGE;
        x.chunk(st, now.unit * UNIT + warp * CHUNK, now.lo, now.pos, 0, 0, lane);
        const Cursor done = now;
        advance(now);
        if (done.unit < done.last && i + 1 < n_units) continue;
        // ---- the pair's end, or the block's.  The next pair's queries are on their way meanwhile; the stage that has just been read
        // takes the warp's sums (its next chunk is asked for behind the second meeting).
        const int rows = rows_of(done), head = head_of(done);
        if (i + 1 < n_units) S::ask_queries(raw, q + ((size_t)now.row * p.nh + head_of(now)) * p.hd, p.hd, rows_of(now), p.hd, lane);
        __syncwarp();
        x.leave(m_s[warp], l_s[warp], reinterpret_cast<float*>(st), lane);
        __syncthreads();
        const bool from_start = began == done.lo / UNIT, to_end = done.unit == done.last;
        float* mine = p.parts + ((size_t)blockIdx.x * 2 + (from_start ? 1 : 0)) * part;
        const unsigned char* sums = smem + (i % S::STAGES) * S::STAGE;
        for (int idx = threadIdx.x; idx < rows * pairs; idx += THREADS) {
            const int r = idx / pairs, d = (idx % pairs) * 2;
            const Joined y = join_warps<S::ROWS, HD>(m_s, l_s, sums, Ring<HD>::WARP, r, d);
            if (from_start && to_end) {
                store_pair(p.out + ((size_t)done.row * p.nh + head + r) * p.hd + d, y.a * inverse(y.l), y.b * inverse(y.l));
            } else {
                *reinterpret_cast<float2*>(mine + r * p.hd + d) = make_float2(y.a, y.b);
                if (d == 0) *reinterpret_cast<float2*>(mine + S::ROWS * p.hd + 2 * r) = make_float2(y.m, y.l);
            }
        }
        if (!(from_start && to_end)) {
            // ---- the last of the pair's blocks to finish joins their parts, in the order of the blocks; where they are many, the
            // last of every PARTS blocks joins theirs first, and the last of all the groups'
            const int each = before[done.row + 1] - before[done.row];
            const long long p0 = (long long)before[done.row] * kv_blocks + (long long)done.kvb * each, p1 = p0 + each - 1;
            // unit u belongs to the last block b with total * b / blocks <= u
            const int b0 = (int)(((p0 + 1) * blocks - 1) / total), b1 = (int)(((p1 + 1) * blocks - 1) / total);
            auto part_of = [&](int b) { return p.parts + ((size_t)b * 2 + (b == b0 ? 1 : 0)) * part; };
            // the parts of the blocks first, first + step, ... (those behind the first aligned to ``step``): to the output or, not
            // normalised, into the first one's place.  Eight parts are on their way at a time.
            auto join_parts = [&](int first, int step, int count, bool to_out) {
                auto nth = [&](int u) { return part_of(u == 0 ? first : first / step * step + u * step); };
                const int quads = p.hd / 4;
                for (int idx = threadIdx.x; idx < rows * quads; idx += THREADS) {
                    const int r = idx / quads, d = idx % quads * 4;
                    float4 got = make_float4(0.f, 0.f, 0.f, 0.f);
                    float most = -INFINITY, sum = 0.f;
                    for (int u0 = 0; u0 < count; u0 += 8) {
                        float4 v[8];
                        float2 ml[8];
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            ml[u] = make_float2(-INFINITY, 0.f);
                            v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (u0 + u < count) {
                                ml[u] = __ldcg(reinterpret_cast<const float2*>(nth(u0 + u) + S::ROWS * p.hd + 2 * r));
                                v[u] = __ldcg(reinterpret_cast<const float4*>(nth(u0 + u) + r * p.hd + d));
                            }
                        }
                        float m8 = most;
#pragma unroll
                        for (int u = 0; u < 8; u++) m8 = fmaxf(m8, ml[u].x);
                        const float f = most == -INFINITY ? (m8 == -INFINITY ? 1.f : 0.f) : exp2_fast(most - m8);
                        sum *= f;
                        got.x *= f, got.y *= f, got.z *= f, got.w *= f;
#pragma unroll
                        for (int u = 0; u < 8; u++) {
                            const float w = ml[u].x == -INFINITY ? 0.f : exp2_fast(ml[u].x - m8);
                            sum += ml[u].y * w;
                            got.x += v[u].x * w, got.y += v[u].y * w, got.z += v[u].z * w, got.w += v[u].w * w;
                        }
                        most = m8;
                    }
                    if (to_out) {
                        const float inv = inverse(sum);
                        bf16* to = p.out + ((size_t)done.row * p.nh + head + r) * p.hd + d;
                        store_pair(to, got.x * inv, got.y * inv);
                        store_pair(to + 2, got.z * inv, got.w * inv);
                    } else {                   // nobody but this thread reads this piece of the first part
                        float* to = part_of(first);
                        *reinterpret_cast<float4*>(to + r * p.hd + d) = got;
                        if (d == 0) joined_ml[r] = make_float2(most, sum);
                    }
                }
                if (!to_out) {                 // (m, l) of the first part are read by all of a row's threads
                    __syncthreads();
                    if (threadIdx.x < rows) *reinterpret_cast<float2*>(part_of(first) + S::ROWS * p.hd + 2 * threadIdx.x) = joined_ml[threadIdx.x];
                }
            };
            // whether this block is the last of ``count`` that come to the counter
            auto am_last = [&](int* c, int count) {
                __syncthreads();
                if (threadIdx.x == 0) {
                    __threadfence();           // the block's parts are there before its count (the fence covers what the barrier has ordered)
                    is_last = atomicAdd(c, 1) == count - 1;
                    if (is_last) *c = 0;
                    __threadfence();
                }
                __syncthreads();
                return is_last != 0;
            };
            int* of_pair = p.counters + (size_t)done.row * kv_blocks + done.kvb;
            if (b1 - b0 < PARTS) {
                if (am_last(of_pair, b1 - b0 + 1)) join_parts(b0, 1, b1 - b0 + 1, true);
            } else {
                const int g = blockIdx.x / PARTS, g0 = b0 / PARTS, g1 = b1 / PARTS, first = max(b0, g * PARTS), last = min(b1, g * PARTS + PARTS - 1);
                // a group's counter: that of its first block, which no other pair's group shares (two slots a block)
                if (am_last(p.counters + (size_t)p.n_rows * kv_blocks + 2 * first + (first == b0 ? 1 : 0), last - first + 1)) {
                    join_parts(first, 1, last - first + 1, false);
                    if (am_last(of_pair, g1 - g0 + 1)) join_parts(b0, PARTS, g1 - g0 + 1, true);
                }
            }
        }
        __syncthreads();                       // the lists and the stages may be written again
        if (i + 1 < n_units) {
            began = now.unit;
            x.begin(raw, p.scale_log2, lane);
        }
    }
    copies_wait<0>();
}

template <typename Kernel> int launch(Kernel kernel, size_t smem, bool (&raised)[64], const Params& p, dim3 grid, cudaStream_t stream) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
    if (!raised[device]) {                                               // per device
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        raised[device] = true;
    }
    esp_launch_pdl(ESP_PDL_ATTENTION, kernel, grid, dim3(THREADS), smem, stream, p);
    return esp_launch_status();
}
template <int HD, int NT> int launch_decode(const Params& p, int blocks, cudaStream_t stream) {
    static bool raised[64] = {false};
    return launch(attn_decode_kv8_kernel<HD, NT>, (size_t)WARPS * Ring<HD>::WARP, raised, p, dim3(blocks), stream);
}
template <int HD> int launch_run(const Params& p, int n_tiles, cudaStream_t stream) {
    static bool raised[64] = {false};
    return launch(attn_run_kv8_kernel<HD, 2>, (size_t)WARPS * Ring<HD>::WARP, raised, p, dim3((unsigned)n_tiles * 8u, p.nh), stream);
}
bool sizes_fit(int nh, int nkv, int hd) { return nkv > 0 && nh > 0 && nh % nkv == 0 && nh <= 65535 && hd > 0 && hd % 8 == 0 && hd <= 256; }
Params make_params(const void* q, const void* k, const void* v, const void* exps, void* out, const int* block_table, int n_seqs, int table_stride, int n_pages, int nh,
                   int nkv, int hd, int window, int* status) {
    Params p{};
    p.q = (const bf16*)q, p.k = (const unsigned char*)k, p.v = (const unsigned char*)v, p.exps = (const unsigned char*)exps, p.out = (bf16*)out;
    p.block_table = block_table, p.n_seqs = n_seqs, p.table_stride = table_stride, p.n_pages = n_pages, p.nh = nh, p.nkv = nkv, p.hd = hd, p.window = window;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
    p.status = status;
    return p;
}
}  // namespace

// One token row of a sequence per row of q.  ``blocks``: the size of the grid, best what the device holds at once.  Scratch: parts
// float [blocks * 2 * 16 * (hd + 2)]; counters int [min(n_tokens, 1024) * nh + 2 * blocks], zero when the call starts and when it ends.  ``seq_past``
// (may be null): per sequence of the step, the positions cached before it.
ESP_API int esp_attn_decode_kv8(const void* q, const void* k, const void* v, const void* exps, void* out, float* parts, int* counters,
                                const int* tok_seq, const int* tok_pos, const int* seq_past, const int* block_table, int n_seqs, int table_stride, int n_pages,
                                int n_tokens, int nh, int nkv, int hd, int window, int blocks, int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (!sizes_fit(nh, nkv, hd) || blocks <= 0 || window < 0 || table_stride <= 0 || table_stride >= (1 << 25) || !parts || !counters)
        return (int)cudaErrorInvalidValue;
    // a launch's units are counted in 32 bits
    if ((long long)(n_tokens < MAX_ROWS ? n_tokens : MAX_ROWS) * (table_stride / 2 + 1) > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    Params p = make_params(q, k, v, exps, out, block_table, n_seqs, table_stride, n_pages, nh, nkv, hd, window, status);
    p.parts = parts, p.counters = counters, p.seq_past = seq_past;
    // The query heads of a key head beyond eight: blocks of sixteen rows, or two of eight, whose keys come from L2 the second time.  Sixteen
    // rows have twice as much to join and, in wide heads, spill; they win where a block has a long way to go (units a block by the
    // page table's width, or by the window where that is less, sixteen rows and eight: 48 heads on 4, 32 sequences of 2,000: 6.9 units, 29.3 and 31.3 us; 28 on 2 of 96
    // channels, 20 of 8,000: 8.4, 30.9 and 36.1; 16 on 1, 20 of 8,000: 4.2, 28.6 and 24.9; 32 on 2, 8 of 4,096: 1.7, 24.0 and 17.5; of 64
    // channels 20 of 8,000: 33.2 and 25.7; 48 on 4 of 256, 8 of 4,096: 56.2 and 40.6; with windows 32 on 2, 64 that see 1,000: 3.4, 26.3 and 22.8;
    // 48 on 4, 32 that see 512: 1.7, 22.6 and 17.7; 28 on 2 of 96 channels, 20 that see 2,000: 2.1, 17.7 and 18.7).
    long long keys = (long long)table_stride * KV8_PAGE;
    if (window > 0 && window < keys) keys = window;
    const bool wide = nh / nkv > 8 && (long long)n_tokens * nkv * keys / UNIT > 5LL * blocks;
    for (int at = 0; at < n_tokens; at += MAX_ROWS) {                    // more rows than a block's list holds: one call behind the other
        p.n_rows = n_tokens - at < MAX_ROWS ? n_tokens - at : MAX_ROWS;
        p.tok_seq = tok_seq + at, p.tok_pos = tok_pos + at;
        p.q = (const bf16*)q + (size_t)at * nh * hd, p.out = (bf16*)out + (size_t)at * nh * hd;
        int rc;
        if (hd <= 64) rc = launch_decode<64, 1>(p, blocks, stream);
        else if (hd <= 96) rc = wide ? launch_decode<96, 2>(p, blocks, stream) : launch_decode<96, 1>(p, blocks, stream);
        else if (hd <= 128) rc = wide ? launch_decode<128, 2>(p, blocks, stream) : launch_decode<128, 1>(p, blocks, stream);
        else if (hd <= 192) rc = launch_decode<192, 1>(p, blocks, stream);
        else rc = launch_decode<256, 1>(p, blocks, stream);
        if (rc) return rc;
    }
    return 0;
}

// Runs of new tokens: tiles of 128 of a sequence (sequence, its first token among the sequence's new ones), of sequences with at
// most ``most`` new tokens (0: of all).  Heads of 72 to 256 channels.
ESP_API int esp_attn_run_kv8(const void* q, long long n_tokens, const void* k, const void* v, const void* exps, void* out, const int* tile_seq,
                             const int* tile_first, const int* seq_start, const int* seq_past, const int* block_table, int n_seqs, int table_stride,
                             int n_pages, int n_tiles, int nh, int nkv, int hd, int window, int most, int* status, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!sizes_fit(nh, nkv, hd) || hd <= 64 || window < 0 || table_stride >= (1 << 25) || n_tiles > (1 << 26) || n_tokens > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    Params p = make_params(q, k, v, exps, out, block_table, n_seqs, table_stride, n_pages, nh, nkv, hd, window, status);
    p.n_rows = (int)n_tokens, p.tile_seq = tile_seq, p.tile_first = tile_first, p.seq_start = seq_start, p.seq_past = seq_past;
    p.most = most > 0 ? most : 0x7fffffff;
    if (hd <= 96) return launch_run<96>(p, n_tiles, stream);
    if (hd <= 128) return launch_run<128>(p, n_tiles, stream);
    return hd <= 192 ? launch_run<192>(p, n_tiles, stream) : launch_run<256>(p, n_tiles, stream);
}
