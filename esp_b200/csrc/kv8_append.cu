// The step's new queries, keys and values on their way from the projection: bias, split-half rotation in 32-bit, queries
// rounded to bfloat16, keys and values rounded into the 8-bit paged cache (kv8.cuh).
//
// qkv: [n_tokens, (nh + 2*nkv) * hd] float, queries, keys, values; ``bias`` (same width, may be null) is added first.
// For i < rot/2 and the token's position p, of queries and keys:
//   o[i]         = x[i] * cos[p][i] - x[i + rot/2] * sin[p][i]
//   o[i + rot/2] = x[i + rot/2] * cos[p][i] + x[i] * sin[p][i]
// Columns at or beyond ``rot`` pass through.  A row's exponent comes from its rotated numbers in 32-bit, so a key is rounded
// once, not to bfloat16 first.
//
// Bound by its launch where there are few tokens, and where there are many by its instructions and by how little it has on its way: short
// blocks that look up position and page first, 73 % of the issue slots.  It is not at the memory's rate, which a copy of as much
// reading as writing shows to be 6.5 TB/s.  A row's lanes hold all of its numbers in registers, so the maximum and the rounding need no
// second pass.  Measured (B200): 8,192 tokens of 48 heads of 128 60 us for 273 MB (4.5 TB/s; a number a lane 300 us), one token 2 to 3 us.
#include "kv8.cuh"

namespace {
struct AppendParams {
    const float *qkv, *bias;
    const int *tok_seq, *tok_pos;
    const float *cos_t, *sin_t;
    int rot, max_pos;
    bf16* q_out;
    unsigned char *k_codes, *v_codes, *exps;
    const int* block_table;
    int n_seqs, table_stride, n_pages, nh, nkv, hd, heads;      // heads: of a token's rows that the call writes (queries alone: nh)
    int* status;
};

// Where the token ``n`` lies: its position (-1: none that has angles) and the page's first row of head 0 (-1: no page).
struct Place {
    int pos;
    long long block;                     // page * nkv, or -1
};
__device__ __forceinline__ Place find_place(const AppendParams& p, int n) {
    Place at{p.tok_pos[n], -1};
    if (at.pos < 0 || (p.rot > 0 && at.pos >= p.max_pos)) {
        at.pos = -1;
    } else if (p.heads > p.nh) {
        const int seq = p.tok_seq[n];
        int page = -1;
        if (at.pos / KV8_PAGE < p.table_stride && seq >= 0 && seq < p.n_seqs) page = p.block_table[(size_t)seq * p.table_stride + at.pos / KV8_PAGE];
        if (page >= 0 && page < p.n_pages) at.block = (long long)page * p.nkv;
    }
    return at;
}
// A key's or value's row: the codes and the exponent of head ``head`` of the projection.
__device__ __forceinline__ unsigned char* row_codes(const AppendParams& p, const Place& at, int head, unsigned char*& exp) {
    const int is_v = head >= p.nh + p.nkv;
    const size_t block = (size_t)(at.block + head - p.nh - (is_v ? p.nkv : 0));
    const int in_page = at.pos % KV8_PAGE;
    exp = p.exps + (block * 2 + is_v) * KV8_PAGE + in_page;
    return (is_v ? p.v_codes : p.k_codes) + (block * KV8_PAGE + in_page) * p.hd;
}

// ``rot`` a multiple of 8: a row is hd / 8 slots of two pieces of four channels, a lane each; ``group`` lanes (a power of two)
// take a row.  The first rot / 8 slots are pairs (i, i + rot/2) that rotate together, the others eight channels that follow one
// another.  Every number is read once, in 16-byte pieces; a thread asks for the pieces of U rows before it looks where they go.
template <int U>
__global__ void __launch_bounds__(256) kv8_append_pairs_kernel(const AppendParams p, int group) {
    pdl_trigger();
    pdl_wait();
    const float* qkv = behind_wait(p.qkv);
    const int rows = blockDim.x / group, slot = threadIdx.x & (group - 1), head0 = blockIdx.y * (rows * U) + threadIdx.x / group;
    if (head0 >= p.heads) return;                        // whole groups; a warp's others go on
    const unsigned mates = group == 32 ? 0xffffffffu : ((1u << group) - 1u) << ((threadIdx.x & 31) & ~(group - 1));
    const bool mine = slot < p.hd / 8, pair = slot < p.rot / 8;
    const int a = pair ? 4 * slot : 8 * slot, b = pair ? a + p.rot / 2 : a + 4;
    const float* token = qkv + (size_t)blockIdx.x * (p.nh + 2 * p.nkv) * p.hd;
    float4 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = head0 + u * rows;
        lo[u] = hi[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (mine && head < p.heads) {
            lo[u] = *reinterpret_cast<const float4*>(token + (size_t)head * p.hd + a);
            hi[u] = *reinterpret_cast<const float4*>(token + (size_t)head * p.hd + b);
        }
    }
    const Place at = find_place(p, blockIdx.x);
    float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (pair && at.pos >= 0) {
        const size_t where = (size_t)at.pos * (p.rot / 2) + a;
        c = *reinterpret_cast<const float4*>(p.cos_t + where);
        s = *reinterpret_cast<const float4*>(p.sin_t + where);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = head0 + u * rows;
        if (head >= p.heads) return;
        if (at.pos < 0 || (head >= p.nh && at.block < 0)) {
            if (slot == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
            continue;
        }
        float4 x = lo[u], y = hi[u];
        if (p.bias && mine) {
            const float4 v = *reinterpret_cast<const float4*>(p.bias + (size_t)head * p.hd + a), w = *reinterpret_cast<const float4*>(p.bias + (size_t)head * p.hd + b);
            x.x += v.x, x.y += v.y, x.z += v.z, x.w += v.w;
            y.x += w.x, y.y += w.y, y.z += w.z, y.w += w.w;
        }
        if (pair && head < p.nh + p.nkv) {
            const float4 v = x, w = y;
            x.x = v.x * c.x - w.x * s.x, y.x = w.x * c.x + v.x * s.x;
            x.y = v.y * c.y - w.y * s.y, y.y = w.y * c.y + v.y * s.y;
            x.z = v.z * c.z - w.z * s.z, y.z = w.z * c.z + v.z * s.z;
            x.w = v.w * c.w - w.w * s.w, y.w = w.w * c.w + v.w * s.w;
        }
        if (head < p.nh) {
            bf16* q = p.q_out + ((size_t)blockIdx.x * p.nh + head) * p.hd;
            if (mine) {
                Vec4<bf16>::store(q + a, x.x, x.y, x.z, x.w);
                Vec4<bf16>::store(q + b, y.x, y.y, y.z, y.w);
            }
            continue;
        }
        // an infinity or a NaN is the largest magnitude when it is looked at as a whole number
        unsigned top = 0;
        auto see = [&](float v) { top = max(top, __float_as_uint(v) & 0x7fffffffu); };
        see(x.x), see(x.y), see(x.z), see(x.w), see(y.x), see(y.y), see(y.z), see(y.w);
        for (int off = group >> 1; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(mates, top, off));
        const int byte = top >= 0x7f800000u ? KV8_NAN : kv8_exponent_byte(__uint_as_float(top));
        const float f = byte == KV8_NAN ? 0.f : kv8_pow2(127 - byte);
        unsigned char *exp, *codes = row_codes(p, at, head, exp);
        if (mine) {
            unsigned v = 0, w = 0;
            if (byte != KV8_NAN) {
                v = kv8_pack2(x.x * f, x.y * f) | kv8_pack2(x.z * f, x.w * f) << 16;
                w = kv8_pack2(y.x * f, y.y * f) | kv8_pack2(y.z * f, y.w * f) << 16;
            }
            *reinterpret_cast<unsigned*>(codes + a) = v;
            *reinterpret_cast<unsigned*>(codes + b) = w;
        }
        if (slot == 0) *exp = (unsigned char)byte;
    }
}

// Any other even ``rot``: a warp a row, lane i holds the numbers i, i + 32, ...
__global__ void __launch_bounds__(256) kv8_append_kernel(AppendParams p) {
    pdl_trigger();
    pdl_wait();
    const float* qkv = behind_wait(p.qkv);
    const int lane = threadIdx.x & 31;
    const int head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (head >= p.heads) return;
    const Place at = find_place(p, blockIdx.x);
    if (at.pos < 0 || (head >= p.nh && at.block < 0)) {
        if (lane == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        return;
    }
    const int half = p.rot / 2;
    const float *x = qkv + ((size_t)blockIdx.x * (p.nh + 2 * p.nkv) + head) * p.hd, *b = p.bias ? p.bias + (size_t)head * p.hd : nullptr;
    const float *cs = p.cos_t + (size_t)at.pos * half, *sn = p.sin_t + (size_t)at.pos * half;
    float v[8];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = j * 32 + lane;
        v[j] = 0.f;
        if (i < p.hd) {
            v[j] = x[i] + (b ? b[i] : 0.f);
            if (i < p.rot && head < p.nh + p.nkv) {
                const int o = i < half ? i + half : i - half, c = i < half ? i : o;
                const float other = x[o] + (b ? b[o] : 0.f);
                v[j] = i < half ? v[j] * cs[c] - other * sn[c] : v[j] * cs[c] + other * sn[c];
            }
            if (head < p.nh) p.q_out[((size_t)blockIdx.x * p.nh + head) * p.hd + i] = __float2bfloat16_rn(v[j]);
        }
        top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
    }
    if (head < p.nh) return;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
    const int byte = top >= 0x7f800000u ? KV8_NAN : kv8_exponent_byte(__uint_as_float(top));
    const float f = byte == KV8_NAN ? 0.f : kv8_pow2(127 - byte);
    unsigned char *exp, *codes = row_codes(p, at, head, exp);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = j * 32 + lane;
        if (i < p.hd) codes[i] = byte == KV8_NAN ? 0 : (unsigned char)kv8_pack2(v[j] * f, 0.f);
    }
    if (lane == 0) *exp = (unsigned char)byte;
}
}  // namespace

// ``write_kv`` 0: queries alone.  Rows whose position has no table row or no page are skipped and the status says so.
ESP_API int esp_kv8_append(const float* qkv, const float* bias, const int* tok_seq, const int* tok_pos, const float* cos_t,
                           const float* sin_t, int rot, int max_pos, void* q_out, void* k_codes, void* v_codes, void* exps,
                           const int* block_table, int n_seqs, int table_stride, int n_pages, int n_tokens, int nh, int nkv, int hd, int write_kv,
                           int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (rot < 0 || rot > hd || (rot & 1) || hd <= 0 || hd % 8 || hd > 256 || nh <= 0 || nkv <= 0 || nh + 2 * nkv > 65535) return (int)cudaErrorInvalidValue;
    const int heads = write_kv ? nh + 2 * nkv : nh;
    const AppendParams p{qkv, bias, tok_seq, tok_pos, cos_t, sin_t, rot, max_pos, (bf16*)q_out, (unsigned char*)k_codes, (unsigned char*)v_codes,
                         (unsigned char*)exps, block_table, n_seqs, table_stride, n_pages, nh, nkv, hd, heads, status};
    if (rot % 8 == 0) {
        int group = 1;
        while (group * 8 < hd) group *= 2;
        // a block holds heads of one token.  Many tokens: small blocks whose threads take three rows each (8,192 tokens of 48 heads of
        // 128: 59 us; 128 threads 61, 256 threads 66, two rows 64, six 73); few: one row a thread, so that there are more blocks.
        const int unroll = n_tokens > 256 ? 3 : 1, most = n_tokens > 256 ? 64 : 256;
        int threads = 32;
        while (threads < most && threads * unroll < heads * group) threads *= 2;
        const int rows = threads / group * unroll;
        const dim3 grid(n_tokens, (heads + rows - 1) / rows);
        if (unroll == 3) esp_launch_pdl(ESP_PDL_SMALL, kv8_append_pairs_kernel<3>, grid, dim3(threads), 0, stream, p, group);
        else esp_launch_pdl(ESP_PDL_SMALL, kv8_append_pairs_kernel<1>, grid, dim3(threads), 0, stream, p, group);
    } else {
        esp_launch_pdl(ESP_PDL_SMALL, kv8_append_kernel, dim3(n_tokens, (heads + 7) / 8), dim3(256), 0, stream, p);
    }
    return esp_launch_status();
}
