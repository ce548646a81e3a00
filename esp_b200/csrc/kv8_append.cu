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
// Bound by memory where there are many tokens (4 bytes read for every one or two written) and by its launch where there are
// few.  A row's lanes hold all of its numbers in registers, so the maximum and the rounding need no second pass.
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
    int table_stride, n_pages, nh, nkv, hd, heads;      // heads: of a token's rows that the call writes (queries alone: nh)
    long long n_rows;                                    // tokens times heads
    int* status;
};

// Where a row of the projection goes.
struct Row {
    const float *x, *b;                  // the row and its bias (or null)
    bool rotates;
    int pos;
    bf16* q;                             // queries; else null
    unsigned char *codes, *exp;          // keys, values; null where the page is not one
    bool live;
};
__device__ __forceinline__ Row find_row(const AppendParams& p, const float* qkv, long long item) {
    Row r;
    const long long n = item / p.heads;
    const int head = (int)(item - n * p.heads);
    r.pos = p.tok_pos[n];
    r.x = qkv + ((size_t)n * (p.nh + 2 * p.nkv) + head) * p.hd;
    r.b = p.bias ? p.bias + (size_t)head * p.hd : nullptr;
    r.rotates = head < p.nh + p.nkv && p.rot > 0;
    r.live = r.pos >= 0 && (p.rot == 0 || r.pos < p.max_pos);
    r.q = nullptr;
    r.codes = r.exp = nullptr;
    if (head < p.nh) {
        r.q = p.q_out + ((size_t)n * p.nh + head) * p.hd;
    } else if (r.live) {
        const int seq = p.tok_seq[n];
        int page = -1;
        if (r.pos / KV8_PAGE < p.table_stride && seq >= 0) page = p.block_table[(size_t)seq * p.table_stride + r.pos / KV8_PAGE];
        if (page < 0 || page >= p.n_pages) {
            r.live = false;
        } else {
            const int is_v = head >= p.nh + p.nkv, kvh = head - p.nh - (is_v ? p.nkv : 0), at = r.pos % KV8_PAGE;
            const size_t block = (size_t)page * p.nkv + kvh;
            r.codes = (is_v ? p.v_codes : p.k_codes) + (block * KV8_PAGE + at) * p.hd;
            r.exp = p.exps + (block * 2 + is_v) * KV8_PAGE + at;
        }
    }
    return r;
}

// A warp a row; any even ``rot``, hd a multiple of 8 up to 256: lane i holds the numbers i, i + 32, ...
__global__ void __launch_bounds__(256) kv8_append_kernel(AppendParams p) {
    pdl_trigger();
    pdl_wait();
    const float* qkv = behind_wait(p.qkv);
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= p.n_rows) return;
    const Row r = find_row(p, qkv, item);
    if (!r.live) {
        if (lane == 0) atomicOr(p.status, ESP_STATUS_BAD_INDEX);
        return;
    }
    const int half = p.rot / 2;
    const float *cs = p.cos_t + (size_t)r.pos * half, *sn = p.sin_t + (size_t)r.pos * half;
    float v[8], amax = 0.f;
    bool fine = true;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = j * 32 + lane;
        v[j] = 0.f;
        if (i < p.hd) {
            v[j] = r.x[i] + (r.b ? r.b[i] : 0.f);
            if (r.rotates && i < p.rot) {
                const int o = i < half ? i + half : i - half, c = i < half ? i : o;
                const float other = r.x[o] + (r.b ? r.b[o] : 0.f);
                v[j] = i < half ? v[j] * cs[c] - other * sn[c] : v[j] * cs[c] + other * sn[c];
            }
            if (r.q) r.q[i] = __float2bfloat16_rn(v[j]);
        }
        fine = fine && isfinite(v[j]);
        amax = fmaxf(amax, fabsf(v[j]));
    }
    if (r.q) return;
    fine = __all_sync(0xffffffffu, fine);
    const int byte = fine ? kv8_exponent_byte(warp_max(amax)) : KV8_NAN;
    const float f = byte == KV8_NAN ? 0.f : kv8_pow2(127 - byte);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = j * 32 + lane;
        if (i < p.hd) r.codes[i] = byte == KV8_NAN ? 0 : (unsigned char)kv8_pack2(v[j] * f, 0.f);
    }
    if (lane == 0) *r.exp = (unsigned char)byte;
}
}  // namespace

// ``write_kv`` 0: queries alone.  Rows whose position has no table row or no page are skipped and the status says so.
ESP_API int esp_kv8_append(const float* qkv, const float* bias, const int* tok_seq, const int* tok_pos, const float* cos_t,
                           const float* sin_t, int rot, int max_pos, void* q_out, void* k_codes, void* v_codes, void* exps,
                           const int* block_table, int table_stride, int n_pages, int n_tokens, int nh, int nkv, int hd, int write_kv,
                           int* status, cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (rot < 0 || rot > hd || (rot & 1) || hd <= 0 || hd % 8 || hd > 256 || nh <= 0 || nkv <= 0) return (int)cudaErrorInvalidValue;
    const int heads = write_kv ? nh + 2 * nkv : nh;
    const AppendParams p{qkv, bias, tok_seq, tok_pos, cos_t, sin_t, rot, max_pos, (bf16*)q_out, (unsigned char*)k_codes, (unsigned char*)v_codes,
                         (unsigned char*)exps, block_table, table_stride, n_pages, nh, nkv, hd, heads, (long long)n_tokens * heads, status};
    const long long blocks = (p.n_rows + 7) / 8;
    if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    esp_launch_pdl(ESP_PDL_SMALL, kv8_append_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return esp_launch_status();
}
