// Attention over the 8-bit paged cache (kv8.cuh), streaming: one new token of every sequence with the keys split over blocks
// (decode), or sixteen new tokens of a run (head sizes that the tensor-memory kernel does not take).
//
//   s_j = q k_j / sqrt(hd),  o = sum_j 2^(s_j log2 e - m) v_j / sum_j 2^(s_j log2 e - m),  m = max_j s_j log2 e
// over the keys max(0, pos - window + 1) <= j <= pos.
//
// A block has four warps and up to 8 * NT rows: the query heads that share one key/value head (decode), or consecutive
// tokens of one head (RUN).  Every warp is on its own until the end: it takes each fourth chunk of 32 keys, brings the
// codes of its chunks in by asynchronous copies (a ring of STAGES chunks, 16 bytes a lane, swizzled so that eight rows of an
// ldmatrix fall into different banks), and keeps a softmax and an output of its own; the warps' and then the splits' results
// are joined in ascending order.
//
// Both products run on mma.sync m16n8k16 in half precision with the cache as the 16-row operand, so a block of up to eight
// rows wastes no more than that: S^T = K Q^T, O^T = V^T P^T.  Codes become halfs exactly by one conversion per two codes
// (through bfloat16 it would be four operations), and the exponents are applied in 32-bit: a key's to its scores, a
// value's to its weight.  A half has little range, so
//   * queries are scaled by a power of two that brings the row's largest to 2^14 (bfloat16's 8 bits fit a half's 11),
//   * the weights 2^(s + e_v) have a running maximum M of their own; the largest weight becomes 2^WEIGHT_TOP and what is
//     rounded off to a half's 11 bits is below 2^-24 of it at most 2^-25 of it.
// Sums, maxima and accumulators are 32-bit.
#include "kv8.cuh"

namespace {
constexpr int THREADS = 128, WARPS = 4, CHUNK = 32;
constexpr float WEIGHT_TOP = 10.f;

struct Params {
    const bf16* q;
    const unsigned char *k, *v, *exps;
    bf16* out;
    float *part_o, *part_ml;
    int* counters;
    const int *tok_seq, *tok_pos;              // decode: per row of the step
    const int *seq_past, *seq_start;           // per sequence (decode: seq_past may be null)
    const int *tile_seq, *tile_first;          // RUN: tiles of tile_rows new tokens
    const int* block_table;
    int table_stride, n_pages, nh, nkv, hd, window, split_keys, n_splits, tile_rows;
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
    static constexpr int STAGES = HD == 64 ? 4 : HD == 128 ? 3 : 2;
    static constexpr int STAGE = CHUNK * HD * 2 + 2 * CHUNK;             // keys, values, exponents of both
    static constexpr int WARP = (STAGES * STAGE + 127) / 128 * 128;
};
// where the 16-byte piece c of row r lies: rows of 64 bytes share 128 bytes with a neighbour
template <int HD> __device__ __forceinline__ int piece_at(int r, int c) {
    return r * HD + ((c ^ (HD == 64 ? (r >> 1) & 3 : r & 7)) << 4);
}

template <int HD, int NT, bool RUN>
__global__ void __launch_bounds__(THREADS) attn_kv8_kernel(const Params p) {
    pdl_trigger();
    constexpr int STAGES = Ring<HD>::STAGES, STAGE = Ring<HD>::STAGE, ROWS = 8 * NT, PP = HD / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float m_s[WARPS][ROWS], l_s[WARPS][ROWS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2, tg = lane & 3;
    unsigned char* ring = smem + warp * Ring<HD>::WARP;

    // ---- the block's rows: ``rows`` of them, row r at query row q0 + r * q_step, at position pos0 + (RUN ? r : 0)
    int seq, kvh, rows, pos0, head0;
    long long q0, q_step;
    if constexpr (RUN) {
        const int subs = p.tile_rows / ROWS, tile = blockIdx.x / subs, first = p.tile_first[tile] + (blockIdx.x % subs) * ROWS;
        seq = p.tile_seq[tile];
        const int start = p.seq_start[seq];
        rows = min(ROWS, p.seq_start[seq + 1] - start - first);
        if (rows <= 0) return;
        head0 = blockIdx.y;
        kvh = head0 / (p.nh / p.nkv);
        pos0 = p.seq_past[seq] + first;
        q0 = (long long)(start + first) * p.nh + head0;
        q_step = p.nh;
    } else {
        const int group = p.nh / p.nkv, per_kv = (group + ROWS - 1) / ROWS;
        kvh = blockIdx.y / per_kv;
        head0 = kvh * group + (blockIdx.y % per_kv) * ROWS;
        rows = min(ROWS, (kvh + 1) * group - head0);
        seq = p.tok_seq[blockIdx.x];
        pos0 = p.tok_pos[blockIdx.x];
        q0 = (long long)blockIdx.x * p.nh + head0;
        q_step = 1;
    }
    const int pos_last = pos0 + (RUN ? rows - 1 : 0);
    if (pos0 < 0 || seq < 0 || pos_last / KV8_PAGE >= p.table_stride) {
        if (threadIdx.x == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        return;
    }
    const int lo = first_visible_key(pos0, p.window, 0);
    const int k0 = RUN ? lo : max(lo, (int)blockIdx.z * p.split_keys);
    const int k1 = RUN ? pos_last : min(pos_last, ((int)blockIdx.z + 1) * p.split_keys - 1);
    if (k0 > k1) return;                       // not one of the row's splits
    const int n_chunks = k1 / CHUNK - k0 / CHUNK + 1, mine = (n_chunks - warp + WARPS - 1) / WARPS;
    const int* pages = p.block_table + (size_t)seq * p.table_stride;
    const bool whole_pieces = p.hd % 16 == 0;

    // ---- copies of this warp's i-th chunk (keys chunk * 32 ..) into a stage; ``page`` was read one chunk ahead
    auto chunk_of = [&](int i) { return k0 / CHUNK + i * WARPS + warp; };
    auto page_of = [&](int i) { return i < mine ? pages[chunk_of(i) * CHUNK / KV8_PAGE] : -1; };
    auto load = [&](int i, int page) {
        if (i < mine) {
            unsigned char* st = ring + (i % STAGES) * STAGE;
            const unsigned k_dst = smem_addr(st), v_dst = k_dst + CHUNK * HD, e_dst = v_dst + CHUNK * HD;
            const int key0 = chunk_of(i) * CHUNK;
            const bool ok = page >= 0 && page < p.n_pages;
            if (!ok && lane == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
            const size_t block = ok ? (size_t)page * p.nkv + kvh : 0;
            const size_t row0 = (block * KV8_PAGE + key0 % KV8_PAGE) * p.hd;
            if (whole_pieces) {
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
            // the exponents: 32 bytes of the keys, 32 of the values (a page that is not one: NaN-free zeros, its keys are hidden)
            if (lane < 16) copy4(e_dst + lane * 4, p.exps + (block * 2 + (lane >> 3)) * KV8_PAGE + key0 % KV8_PAGE + (lane & 7) * 4, ok ? 4 : 0);
        }
        copies_commit();
    };
    // Positions that were cached before this step do not depend on the kernel before this one, which writes the step's
    // own: a decode block all of whose keys are older asks for its first chunks at once and then waits for the queries.
    const bool early = !RUN && p.seq_past != nullptr && k1 < p.seq_past[seq];
    if (!early) pdl_wait();
    int page_next = page_of(0);
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) {
        const int page = page_next;
        page_next = page_of(s + 1);
        load(s, page);
    }
    if (early) pdl_wait();

    // ---- the queries as B operands, scaled row by row; row_scale: what a score is multiplied by (before the key's exponent)
    const bf16* q = behind_wait(p.q);
    unsigned qf[NT][HD / 16][2];
    float row_scale[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = nt * 8 + g8;
        const bf16* row = q + (q0 + r * q_step) * p.hd;
        float amax = 0.f;
        uint2 raw[HD / 16];
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
            const int d = kk * 16 + tg * 4;
            raw[kk] = r < rows && d < p.hd ? *reinterpret_cast<const uint2*>(row + d) : make_uint2(0u, 0u);
            const float2 a = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].x)), b = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].y));
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int x = max((int)(__float_as_uint(amax) >> 23) - 127, -100);       // the largest lies in [2^x, 2^(x+1))
        const float f = kv8_pow2(14 - x);
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++) {
            const float2 a = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].x)), b = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].y));
            qf[nt][kk][0] = pack_half(a.x * f, a.y * f);
            qf[nt][kk][1] = pack_half(b.x * f, b.y * f);
        }
        // a lane's scores belong to rows 2 tg and 2 tg + 1, whose queries the lanes 8 tg and 8 tg + 4 hold
        const int xa = __shfl_sync(0xffffffffu, x, tg * 8), xb = __shfl_sync(0xffffffffu, x, tg * 8 + 4);
        row_scale[nt][0] = kv8_pow2(min(xa - 14, 127)) * p.scale_log2;
        row_scale[nt][1] = kv8_pow2(min(xb - 14, 127)) * p.scale_log2;
    }

    float o[NT][HD / 16][4], m[NT][2], l[NT][2], top[NT][2];             // top: M, the running maximum of the weights' exponents
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
        for (int i = 0; i < HD / 16; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) o[nt][i][j] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            m[nt][j] = top[nt][j] = -INFINITY;
            l[nt][j] = 0.f;
        }
    }

    for (int i = 0; i < mine; i++) {
        copies_wait<STAGES - 2>();
        __syncwarp();                          // every lane's pieces of chunk i are there, and all have read chunk i - 1
        {
            const int page = page_next;
            page_next = page_of(i + STAGES);
            load(i + STAGES - 1, page);
        }
        const unsigned char* st = ring + (i % STAGES) * STAGE;
        const unsigned k_src = smem_addr(st), v_src = k_src + CHUNK * HD;
        const unsigned char* e_src = st + 2 * CHUNK * HD;
        const int key0 = chunk_of(i) * CHUNK;
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
            kf[u] = ke == KV8_NAN || vb == KV8_NAN ? __int_as_float(0x7fffffff) : __uint_as_float((unsigned)ke << 23);
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
                    float x = s[nt][u >> 1][(u & 1) * 2 + j] * row_scale[nt][j] * kf[u];
                    bool live = seen[u];
                    if constexpr (RUN) {
                        const int key = key0 + u * 8 + g8, pos = pos0 + nt * 8 + 2 * tg + j;
                        live = live && key <= pos && (p.window <= 0 || pos - key < p.window);
                    }
                    if (!live) x = -INFINITY;
                    s[nt][u >> 1][(u & 1) * 2 + j] = x;
                    t[u][j] = x + ve[u];
                    cm[j] = fmaxf(cm[j], x);
                    ct[j] = fmaxf(ct[j], t[u][j]);
                }
            float mu[2], tu[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    cm[j] = fmaxf(cm[j], __shfl_xor_sync(0xffffffffu, cm[j], off));
                    ct[j] = fmaxf(ct[j], __shfl_xor_sync(0xffffffffu, ct[j], off));
                }
                cm[j] = fmaxf(m[nt][j], cm[j]);
                ct[j] = fmaxf(top[nt][j], ct[j]);
                mu[j] = cm[j] == -INFINITY ? 0.f : cm[j];
                tu[j] = ct[j] == -INFINITY ? 0.f : ct[j];
                l[nt][j] *= exp2_fast(m[nt][j] - mu[j]);
                m[nt][j] = cm[j];
            }
            if (__any_sync(0xffffffffu, ct[0] > top[nt][0] || ct[1] > top[nt][1])) {
                const float a = exp2_fast(top[nt][0] - tu[0]), b = exp2_fast(top[nt][1] - tu[1]);
#pragma unroll
                for (int d = 0; d < HD / 16; d++) {
                    o[nt][d][0] *= a;
                    o[nt][d][1] *= b;
                    o[nt][d][2] *= a;
                    o[nt][d][3] *= b;
                }
                top[nt][0] = ct[0];
                top[nt][1] = ct[1];
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                float w[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    l[nt][j] += exp2_fast(s[nt][u >> 1][(u & 1) * 2 + j] - mu[j]);
                    w[j] = exp2_fast(t[u][j] - tu[j] + WEIGHT_TOP);
                }
                wf[nt][u] = transpose_8x8(pack_half(w[0], w[1]));
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
    copies_wait<0>();
    __syncwarp();

    // ---- the warp's result in the form (m, l, sum of weights 2^(s - m) times values), into its part of shared memory
    float* o_w = reinterpret_cast<float*>(ring);                         // [ROWS][HD]
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
            float sum = l[nt][j];
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            const int r = nt * 8 + 2 * tg + j;
            const float f = m[nt][j] == -INFINITY ? 1.f : exp2_fast(top[nt][j] - WEIGHT_TOP - m[nt][j]);
            if (g8 == 0) {
                m_s[warp][r] = m[nt][j];
                l_s[warp][r] = sum;
            }
#pragma unroll
            for (int d = 0; d < HD / 16; d++)
                *reinterpret_cast<float2*>(o_w + r * HD + d * 16 + 2 * g8) = make_float2(o[nt][d][j] * f, o[nt][d][j + 2] * f);
        }
    __syncthreads();
    // ---- the warps in ascending order.  A warp that saw nothing has m = -inf, l = 0, o = 0; one that saw only rows that are not
    // numbers has m = -inf and NaN in l and o, which stay (0 * NaN = NaN).
    const int first_split = lo / p.split_keys, n_live = RUN ? 1 : pos_last / p.split_keys - first_split + 1;
    auto join = [&](int r, float (&w)[WARPS], float& mx, float& sum) {
        mx = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int u = 0; u < WARPS; u++) mx = fmaxf(mx, m_s[u][r]);
#pragma unroll
        for (int u = 0; u < WARPS; u++) {
            w[u] = m_s[u][r] == -INFINITY ? 0.f : exp2_fast(m_s[u][r] - mx);
            sum += l_s[u][r] * w[u];
        }
    };
    // the sum is 0 where none of the row's pages was one
    auto inverse = [](float sum) { return sum == 0.f ? 0.f : 1.f / sum; };
    const int pairs = p.hd / 2;
    for (int idx = threadIdx.x; idx < rows * pairs; idx += THREADS) {
        const int r = idx / pairs, d = (idx % pairs) * 2;
        float w[WARPS], mx, sum, a = 0.f, b = 0.f;
        join(r, w, mx, sum);
#pragma unroll
        for (int u = 0; u < WARPS; u++) {
            const float2 x = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(smem + u * Ring<HD>::WARP) + r * HD + d);
            a += x.x * w[u];
            b += x.y * w[u];
        }
        if (n_live == 1) {
            const float inv = inverse(sum);
            *reinterpret_cast<__nv_bfloat162*>(p.out + (q0 + r * q_step) * p.hd + d) = __floats2bfloat162_rn(a * inv, b * inv);
        } else {
            const size_t at = ((size_t)blockIdx.x * p.nh + head0 + r) * p.n_splits + blockIdx.z;
            *reinterpret_cast<float2*>(p.part_o + at * p.hd + d) = make_float2(a, b);
            if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(mx, sum);
        }
    }
    if constexpr (RUN) return;
    if (n_live == 1) return;
    // ---- the last block of the row to finish joins its splits, in ascending order
    __shared__ int is_last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int* c = p.counters + (size_t)blockIdx.x * gridDim.y + blockIdx.y;
        is_last = atomicAdd(c, 1) == n_live - 1;
        if (is_last) *c = 0;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    constexpr int AT_ONCE = Ring<HD>::WARP / 8;                          // splits whose weights a warp holds at a time
    float *w_w = reinterpret_cast<float*>(ring), *l_w = w_w + AT_ONCE;
    constexpr int NV = HD / 64;                                          // pairs of channels a lane: 64 j + 2 lane
    for (int r = warp; r < rows; r += WARPS) {
        const size_t at = ((size_t)blockIdx.x * p.nh + head0 + r) * p.n_splits + first_split;
        const float *ml = p.part_ml + at * 2, *po = p.part_o + at * p.hd;
        float mx = -INFINITY, sum = 0.f, num[NV][2];
        for (int i = lane; i < n_live; i += 32) mx = fmaxf(mx, __ldcg(ml + 2 * i));
        mx = warp_max(mx);
#pragma unroll
        for (int j = 0; j < NV; j++) num[j][0] = num[j][1] = 0.f;
        for (int c0 = 0; c0 < n_live; c0 += AT_ONCE) {
            const int cn = min(AT_ONCE, n_live - c0);
            __syncwarp();
            for (int i = lane; i < cn; i += 32) {
                const float2 v = __ldcg(reinterpret_cast<const float2*>(ml + 2 * (c0 + i)));
                w_w[i] = v.x == -INFINITY ? 0.f : exp2_fast(v.x - mx);
                l_w[i] = v.y;
            }
            __syncwarp();
#pragma unroll 8
            for (int i = 0; i < cn; i++) {
                const float w = w_w[i];
                sum += l_w[i] * w;
#pragma unroll
                for (int j = 0; j < NV; j++)
                    if (j * 64 + 2 * lane < p.hd) {
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(po + (size_t)(c0 + i) * p.hd + j * 64 + 2 * lane));
                        num[j][0] += v.x * w;
                        num[j][1] += v.y * w;
                    }
            }
        }
        const float inv = inverse(sum);
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (j * 64 + 2 * lane < p.hd)
                *reinterpret_cast<__nv_bfloat162*>(p.out + (q0 + r) * p.hd + j * 64 + 2 * lane) = __floats2bfloat162_rn(num[j][0] * inv, num[j][1] * inv);
    }
}

template <int HD, int NT, bool RUN> int launch(const Params& p, dim3 grid, cudaStream_t stream) {
    const size_t smem = (size_t)WARPS * Ring<HD>::WARP;
    static bool raised[64] = {false};                                    // per device
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return (int)cudaErrorInvalidDevice;
    if (!raised[device]) {
        const cudaError_t e = cudaFuncSetAttribute(attn_kv8_kernel<HD, NT, RUN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        raised[device] = true;
    }
    esp_launch_pdl(ESP_PDL_ATTENTION, attn_kv8_kernel<HD, NT, RUN>, grid, dim3(THREADS), smem, stream, p);
    return esp_launch_status();
}
template <int NT, bool RUN> int launch_size(const Params& p, dim3 grid, cudaStream_t stream) {
    if (p.hd <= 64) return launch<64, NT, RUN>(p, grid, stream);
    if (p.hd <= 128) return launch<128, NT, RUN>(p, grid, stream);
    return launch<256, NT, RUN>(p, grid, stream);
}
bool sizes_fit(int nh, int nkv, int hd) { return nkv > 0 && nh > 0 && nh % nkv == 0 && nh <= 65535 && hd > 0 && hd % 8 == 0 && hd <= 256; }
}  // namespace

// One token row of the step per block row.  ``split``: key positions a block, a multiple of 64; n_splits * split covers
// the longest row.  Where n_splits > 1: scratch float [n_tokens * nh * n_splits * (hd + 2)], counters
// int [n_tokens * nh], zero when the call starts and when it ends.  ``seq_past`` (may be null): per sequence
// of the step, the positions cached before it.
ESP_API int esp_attn_decode_kv8(const void* q, const void* k, const void* v, const void* exps, void* out, float* scratch, int* counters,
                                const int* tok_seq, const int* tok_pos, const int* seq_past, const int* block_table,
                                int table_stride, int n_pages, int n_tokens, int nh, int nkv, int hd, int window, int split, int n_splits,
                                int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (!sizes_fit(nh, nkv, hd) || n_splits <= 0 || n_splits > 65535 || split < KV8_PAGE || split % KV8_PAGE || window < 0 ||
        (n_splits > 1 && (!scratch || !counters)) || (long long)split * n_splits < (long long)table_stride * KV8_PAGE)
        return (int)cudaErrorInvalidValue;
    Params p{};
    p.q = (const bf16*)q, p.k = (const unsigned char*)k, p.v = (const unsigned char*)v, p.exps = (const unsigned char*)exps, p.out = (bf16*)out;
    p.part_o = scratch, p.part_ml = scratch ? scratch + (size_t)n_tokens * nh * n_splits * hd : nullptr, p.counters = counters, p.tok_seq = tok_seq, p.tok_pos = tok_pos, p.seq_past = seq_past;
    p.block_table = block_table, p.table_stride = table_stride, p.n_pages = n_pages, p.nh = nh, p.nkv = nkv, p.hd = hd, p.window = window;
    p.split_keys = split, p.n_splits = n_splits, p.status = status;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
    const int group = nh / nkv;
    if (group <= 8) return launch_size<1, false>(p, dim3(n_tokens, nkv, n_splits), stream);
    return launch_size<2, false>(p, dim3(n_tokens, nkv * ((group + 15) / 16), n_splits), stream);
}

// Runs of new tokens: tiles of 128 of a sequence (sequence, its first token among the sequence's new ones).
ESP_API int esp_attn_run_kv8(const void* q, const void* k, const void* v, const void* exps, void* out, const int* tile_seq,
                             const int* tile_first, const int* seq_start, const int* seq_past, const int* block_table, int table_stride,
                             int n_pages, int n_tiles, int nh, int nkv, int hd, int window, int* status, cudaStream_t stream) {
    if (n_tiles <= 0) return 0;
    if (!sizes_fit(nh, nkv, hd) || window < 0 || n_tiles > (1 << 26)) return (int)cudaErrorInvalidValue;
    Params p{};
    p.q = (const bf16*)q, p.k = (const unsigned char*)k, p.v = (const unsigned char*)v, p.exps = (const unsigned char*)exps, p.out = (bf16*)out;
    p.tile_seq = tile_seq, p.tile_first = tile_first, p.seq_start = seq_start, p.seq_past = seq_past;
    p.block_table = block_table, p.table_stride = table_stride, p.n_pages = n_pages, p.nh = nh, p.nkv = nkv, p.hd = hd, p.window = window;
    p.split_keys = 1 << 30, p.n_splits = 1, p.tile_rows = 128, p.status = status;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)hd));
    return launch_size<2, true>(p, dim3((unsigned)n_tiles * 8u, nh), stream);
}
