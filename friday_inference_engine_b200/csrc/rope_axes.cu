// Rotary positions with several axes: pair i of a head turns by positions[row][a(i)] / denom[i], where a(i) is the axis (time,
// height, width) that the pair's section belongs to.  Two operations share the kernel:
//
//   rotate   `heads` heads of every row of x -> out (the same place or another)
//   append   a row is [queries | keys | values]: queries -> q_out turned, keys -> the cache's pages turned, values -> pages as they
//            are.  The place in the cache (row_seq, row_pos) and the positions that turn the heads are different numbers here, which
//            is what sets this apart from rowwise.cu's rope_kv_write: all tokens of an image share a time position.
//
// Angles.  A turn is 2^64: a pair's step per position is kept as a 64-bit fraction of a turn, 2^64 / (2 pi denom), formed in double
// precision; position times step modulo 2^64 is then exactly the angle's fraction of a turn for every 32-bit position (a float
// division leaves an error of pos * 2^-24, which at position 10^6 is 0.06 rad).  The upper 32 bits go through sincospif.
#include <math.h>

#include "common.cuh"

FR_EXPORT const char* rope_axes_last_error() { return fr_error_text; }

namespace {

constexpr int MOST_AXES = 4;
constexpr int MOST_HALF = 128;            // pairs of a head that turn: head sizes up to 256

struct RopeArgs {
    const void* x;                        // rows of ld elements
    void* out;                            // turned heads 0 .. nq - 1, rows of out_ld elements
    const int* positions;                 // [rows][axes]
    const float* denom;                   // [half]
    const int* row_seq;                   // null: every row counts (rotate)
    const int* row_pos;
    const int* block_table;
    void* k_pool;
    void* v_pool;
    long long ld, out_ld;
    int rows, nq, nkv, hd, half, axes, interleaved, neighbours;
    int section_end[MOST_AXES];           // pairs of the axes up to and with this one (chunked), or the section itself (interleaved)
    int n_seqs, table_width, page, pool_pages;
};

// the axis that turns pair i
__device__ __forceinline__ int axis_of(const RopeArgs& p, int i) {
    if (p.interleaved) {
        const int a = i % p.axes;
        return i < p.axes * p.section_end[a] ? a : 0;
    }
    int a = 0;
    while (a + 1 < p.axes && i >= p.section_end[a]) ++a;
    return a;
}

// the step per position of a pair, in units of 2^-64 turns
__device__ __forceinline__ unsigned long long turn_step(float denom) {
    const double turns = 0.15915494309189533577 / (double)denom;           // 1 / (2 pi)
    const double frac = turns - rint(turns);                               // [-1/2, 1/2]
    return (unsigned long long)(long long)(frac * 9223372036854775808.0) << 1;
}

__device__ __forceinline__ void sin_cos_at(unsigned long long step, int pos, float& s, float& c) {
    const unsigned long long turn = step * (unsigned long long)(long long)pos;
    sincospif((float)(int)(turn >> 32) * (1.0f / 2147483648.0f), &s, &c);
}

// where the cache keeps (sequence, position); -1: nowhere (a position that the table does not name)
__device__ __forceinline__ long long cache_row(const RopeArgs& p, int seq, int pos) {
    if (seq < 0 || seq >= p.n_seqs || pos < 0 || pos / p.page >= p.table_width) return -1;
    const int pg = p.block_table[(size_t)seq * p.table_width + pos / p.page];
    if (pg < 0 || pg >= p.pool_pages) return -1;
    return (long long)pg * p.page + pos % p.page;
}

template <typename T>
__global__ void __launch_bounds__(256) rope_axes_kernel(const RopeArgs p) {
    __shared__ float2 cs[MOST_HALF];
    fr_pdl_wait();
    fr_pdl_launch();
    const int row = blockIdx.x;
    const int seq = p.row_seq != nullptr ? p.row_seq[row] : 0;
    if (seq < 0) return;
    for (int i = threadIdx.x; i < p.half; i += blockDim.x) {
        float s, c;
        sin_cos_at(turn_step(p.denom[i]), p.positions[(size_t)row * p.axes + axis_of(p, i)], s, c);
        cs[i] = make_float2(c, s);
    }
    __syncthreads();
    const long long at = p.nkv > 0 ? cache_row(p, seq, p.row_pos[row]) : -1;
    const T* x = (const T*)p.x + (size_t)row * p.ld;
    const int heads = p.nq + 2 * p.nkv;
    for (int idx = threadIdx.x; idx < heads * p.hd; idx += blockDim.x) {
        const int h = idx / p.hd, d = idx - h * p.hd;
        T* dst;
        if (h < p.nq) {
            dst = (T*)p.out + (size_t)row * p.out_ld + (size_t)h * p.hd;
        } else {
            if (at < 0) break;
            const int kh = h < p.nq + p.nkv ? h - p.nq : h - p.nq - p.nkv;
            dst = (T*)(h < p.nq + p.nkv ? p.k_pool : p.v_pool) + ((size_t)at * p.nkv + kh) * p.hd;
        }
        const T* src = x + (size_t)h * p.hd;
        if (h >= p.nq + p.nkv || d >= 2 * p.half) {
            dst[d] = src[d];
            continue;
        }
        // the thread of a pair's first number writes both
        const bool first = p.neighbours ? (d & 1) == 0 : d < p.half;
        if (!first) continue;
        const int i = p.neighbours ? d >> 1 : d, e = p.neighbours ? d + 1 : d + p.half;
        float a, b;
        fr_rotate(fr_load(src + d), fr_load(src + e), cs[i].x, cs[i].y, a, b);
        fr_store(dst + d, a);
        fr_store(dst + e, b);
    }
}

int check(const RopeArgs& p, int dtype, const int* sections) {
    if (dtype != FR_F32 && dtype != FR_BF16) FR_REFUSE("rope_axes: unknown dtype %d", dtype);
    if (p.axes < 1 || p.axes > MOST_AXES) FR_REFUSE("rope_axes: %d axes (1 to %d)", p.axes, MOST_AXES);
    if (p.hd < 1 || p.nq < 0 || p.nkv < 0 || p.nq + p.nkv < 1) FR_REFUSE("rope_axes: %d heads, %d kv heads of %d numbers", p.nq, p.nkv, p.hd);
    for (int a = 0; a < p.axes; ++a)
        if (sections[a] < 0 || sections[a] > MOST_HALF) FR_REFUSE("rope_axes: a section of %d pairs", sections[a]);
    if (p.half < 1 || p.half > MOST_HALF || 2 * p.half > p.hd)
        FR_REFUSE("rope_axes: sections of %d pairs in all do not fit heads of %d numbers (and %d pairs are the most)", p.half, p.hd, MOST_HALF);
    if (p.interleaved)
        for (int a = 1; a < p.axes; ++a)
            if (sections[a] > 0 && p.axes * (sections[a] - 1) + a >= p.half)
                FR_REFUSE("rope_axes: axis %d has %d pairs, more than its turns among %d pairs of %d axes", a, sections[a], p.half, p.axes);
    return FR_OK;
}

int launch(RopeArgs& p, const int* sections, int dtype, cudaStream_t stream) {
    p.half = 0;
    for (int a = 0; a < p.axes && a < MOST_AXES; ++a) {
        p.half += sections[a];
        p.section_end[a] = p.interleaved ? sections[a] : p.half;
    }
    const int rc = check(p, dtype, sections);
    if (rc || p.rows <= 0) return rc;
    if (dtype == FR_F32) FR_CUDA(fr_launch(rope_axes_kernel<float>, dim3(p.rows), dim3(256), 0, stream, p));
    else FR_CUDA(fr_launch(rope_axes_kernel<__nv_bfloat16>, dim3(p.rows), dim3(256), 0, stream, p));
    FR_CHECK_LAUNCH("rope_axes");
    return FR_OK;
}

}  // namespace

// x: rows of ld elements, head h at h * hd; out likewise (out == x with the same row length: in place).  positions [rows][axes];
// denom [sum of sections]; sections: host, [axes].
FR_EXPORT int rope_axes_rotate(const void* x, long long ld, void* out, long long out_ld, int rows, int heads, int hd, const int* positions,
                               int axes, const float* denom, const int* sections, int interleaved, int neighbours, int dtype,
                               cudaStream_t stream) {
    RopeArgs p = {};
    p.x = x; p.ld = ld; p.out = out; p.out_ld = out_ld; p.rows = rows; p.nq = heads; p.hd = hd; p.positions = positions; p.axes = axes;
    p.denom = denom; p.interleaved = interleaved != 0; p.neighbours = neighbours != 0;
    return launch(p, sections, dtype, stream);
}

// qkv: rows of ld elements, [nq | nkv | nkv] heads of hd.  Rows whose row_seq is negative are left alone (their queries too); a row
// whose place the table does not name (a position beyond it, a negative page, a page beyond the pool) only gets its queries.
FR_EXPORT int rope_axes_append(const void* qkv, long long ld, void* q_out, long long q_ld, int rows, int nq, int nkv, int hd,
                               const int* row_seq, const int* row_pos, const int* positions, int axes, const float* denom,
                               const int* sections, int interleaved, int neighbours, void* k_pool, void* v_pool, int pool_pages, int page,
                               const int* block_table, int n_seqs, int table_width, int dtype, cudaStream_t stream) {
    RopeArgs p = {};
    if (nkv < 1 || page < 1 || table_width < 1 || n_seqs < 1 || pool_pages < 1)
        FR_REFUSE("rope_axes: a cache of %d pages of %d rows, %d kv heads, a table of %d x %d", pool_pages, page, nkv, n_seqs, table_width);
    p.x = qkv; p.ld = ld; p.out = q_out; p.out_ld = q_ld; p.rows = rows; p.nq = nq; p.nkv = nkv; p.hd = hd; p.row_seq = row_seq;
    p.row_pos = row_pos; p.positions = positions; p.axes = axes; p.denom = denom; p.interleaved = interleaved != 0;
    p.neighbours = neighbours != 0; p.k_pool = k_pool; p.v_pool = v_pool; p.pool_pages = pool_pages; p.page = page;
    p.block_table = block_table; p.n_seqs = n_seqs; p.table_width = table_width;
    return launch(p, sections, dtype, stream);
}
