// Causal grouped-query attention of a batch whose sequences share a long prefix.
//
// The prefix' keys and values lie in pages that one table names for all sequences (prefix_table); what a sequence has behind the
// prefix lies in its own pages (its row of block_table).  Position j of a sequence is prefix key j for j < L and its own key j - L
// from there on; the two ranges' pages are apart, so a prefix may end anywhere in its last page.  A row at position p sees position
// j iff p - window < j <= p (window 0: all j <= p) and a table names room for it; a page that a table leaves out (negative, or
// beyond the pool) reads as zeros.  A row that sees nothing gives zeros; a row whose row_seq is negative, or not below n_seqs, is
// not written.
//
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q . k_j - m),  m = max_j scale q . k_j
//
// Any split of the keys gives partial (m, l = sum w, o = sum w v), and parts join exactly: with M = max m_s,
// out = sum_s o_s exp(m_s - M) / sum_s l_s exp(m_s - M).
#include <math.h>

#include "common.cuh"

FR_EXPORT const char* attention_shared_last_error() { return fr_error_text; }

namespace {

typedef __nv_bfloat16 bf16;
constexpr int MOST_HEAD = 256;
constexpr int MOST_PARTS = 64;

struct SharedArgs {
    const void* q;            // rows of q_stride elements, head h at h * hd
    void* out;                // [rows][nq * hd]
    const void* k_pool;       // [pool_pages][page][nkv][hd]
    const void* v_pool;
    const int* prefix_table;  // [ceil(L / page)]
    const int* block_table;   // [n_seqs][table_width]
    const int* row_seq;       // [rows]
    const int* row_pos;       // [rows]
    float* part;              // [rows * nq][parts][hd]: o
    float* stat;              // [rows * nq][parts][2]: m (in units of log2), l
    long long q_stride;
    int rows, n_seqs, nq, nkv, hd, window, prefix, page, pool_pages, table_width, parts;
    float scale_log2;         // scale times log2(e)
};

// the pool's row of position j of sequence `seq`; -1: no page is named
__device__ __forceinline__ long long place_of(const SharedArgs& p, int seq, int j) {
    const bool shared = j < p.prefix;
    const int k = shared ? j : j - p.prefix;
    const int pg = shared ? p.prefix_table[k / p.page] : p.block_table[(size_t)seq * p.table_width + k / p.page];
    return pg < 0 || pg >= p.pool_pages ? -1 : (long long)pg * p.page + k % p.page;
}

// ------------------------------------------------------------------ every type and head size
// A warp owns one (row, head, part) and walks its share of the keys with a running maximum and sum, the head's numbers spread over
// the lanes.
template <typename T, int PER_LANE>
__global__ void __launch_bounds__(128) rows_kernel(const SharedArgs p) {
    fr_pdl_wait();
    fr_pdl_launch();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long)p.rows * p.nq) return;
    const int row = (int)(item / p.nq), h = (int)(item - (long long)row * p.nq);
    const int seq = p.row_seq[row];
    if (seq < 0 || seq >= p.n_seqs) return;
    const int pos = p.row_pos[row];
    const long long room = (long long)p.prefix + (long long)p.table_width * p.page;
    const int hi = (int)min((long long)pos, room - 1);                     // the last position it sees, and the first
    const int lo = fr_first_key(pos, p.window, 0);
    const int n = hi >= lo ? hi - lo + 1 : 0, share = (n + p.parts - 1) / p.parts;
    const int j0 = lo + (int)min((long long)n, (long long)share * blockIdx.y), j1 = (int)min((long long)lo + n, (long long)j0 + share);
    float qv[PER_LANE], acc[PER_LANE];
    const T* q = (const T*)p.q + (size_t)row * p.q_stride + (size_t)h * p.hd;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int d = lane + 32 * i;
        qv[i] = d < p.hd ? fr_load(q + d) * p.scale_log2 : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int kvh = h / (p.nq / p.nkv);
    for (int j = j0; j < j1; ++j) {
        const long long at = place_of(p, seq, j);
        const size_t base = ((size_t)max(at, 0ll) * p.nkv + kvh) * p.hd;
        float s = 0.f, v[PER_LANE];
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int d = lane + 32 * i;
            const bool there = d < p.hd && at >= 0;
            if (there) s = fmaf(qv[i], fr_load((const T*)p.k_pool + base + d), s);
            v[i] = there ? fr_load((const T*)p.v_pool + base + d) : 0.f;
        }
        s = fr_warp_sum(s);
        const float big = fmaxf(m, s);
        // (a score of -infinity before any other: nothing yet, and no difference of infinities)
        const float keep = m == -INFINITY ? 0.f : exp2f(m - big), w = s == -INFINITY ? 0.f : exp2f(s - big);
        l = l * keep + w;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) acc[i] = fmaf(w, v[i], acc[i] * keep);
        m = big;
    }
    if (p.parts == 1) {
        const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;          // (a NaN stays one)
        T* out = (T*)p.out + ((size_t)row * p.nq + h) * p.hd;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (lane + 32 * i < p.hd) fr_store(out + lane + 32 * i, acc[i] * inv);
        return;
    }
    const size_t mine = (size_t)item * p.parts + blockIdx.y;
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i)
        if (lane + 32 * i < p.hd) p.part[mine * p.hd + lane + 32 * i] = acc[i];
    if (lane == 0) {
        p.stat[2 * mine] = m;
        p.stat[2 * mine + 1] = l;
    }
}

// ------------------------------------------------------------------ joining the parts
// A warp per (row, head).  A part that saw no key has l = 0 and drops out; its o is not read.
template <typename T>
__global__ void __launch_bounds__(128) merge_kernel(const SharedArgs p) {
    fr_pdl_wait();
    fr_pdl_launch();
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long)p.rows * p.nq) return;
    const int row = (int)(item / p.nq);
    const int seq = p.row_seq[row];
    if (seq < 0 || seq >= p.n_seqs) return;
    // lane s has the statistics of parts s and s + 32
    const float* stat = p.stat + 2 * (size_t)item * p.parts;
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool there = lane + 32 * i < p.parts;
        m[i] = there ? stat[2 * (lane + 32 * i)] : -INFINITY;
        l[i] = there ? stat[2 * (lane + 32 * i) + 1] : 0.f;
        if (l[i] == 0.f) m[i] = -INFINITY;
    }
    const float big = fr_warp_max(fmaxf(m[0], m[1]));
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) f[i] = l[i] == 0.f ? 0.f : exp2f(m[i] - big);
    const float sum = fr_warp_sum(f[0] * l[0] + f[1] * l[1]);
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    float acc[MOST_HEAD / 32];
#pragma unroll
    for (int i = 0; i < MOST_HEAD / 32; ++i) acc[i] = 0.f;
    for (int s = 0; s < p.parts; ++s) {
        const float w = __shfl_sync(0xffffffffu, s < 32 ? f[0] : f[1], s & 31);
        if (w == 0.f) continue;
        const float* o = p.part + ((size_t)item * p.parts + s) * p.hd;
#pragma unroll
        for (int i = 0; i < MOST_HEAD / 32; ++i)
            if (lane + 32 * i < p.hd) acc[i] = fmaf(w, o[lane + 32 * i], acc[i]);
    }
    T* out = (T*)p.out + (size_t)item * p.hd;
#pragma unroll
    for (int i = 0; i < MOST_HEAD / 32; ++i)
        if (lane + 32 * i < p.hd) fr_store(out + lane + 32 * i, acc[i] * inv);
}

// ------------------------------------------------------------------ host side
struct Plan {
    int parts = 1;
};

// Keys a row may see in all, at most.
long long reach_of(int max_kv_len, int window) { return window > 0 && window < max_kv_len ? window : max_kv_len; }

// Warps for two rounds of the device's, with at least 64 keys each.
Plan plan_of(long long rows, int nq, int max_kv_len, int window) {
    Plan plan;
    const int sms = fr_sm_count();
    const long long warps = rows * nq, want = 32ll * (sms > 0 ? sms : 128), most = (reach_of(max_kv_len, window) + 63) / 64;
    long long parts = warps > 0 ? want / warps : 1;
    if (parts > most) parts = most;
    plan.parts = (int)(parts < 1 ? 1 : parts > MOST_PARTS ? MOST_PARTS : parts);
    return plan;
}

long long floats_of(const Plan& plan, long long rows, int nq, int hd) { return plan.parts > 1 ? rows * nq * plan.parts * (hd + 2) : 0; }

template <typename T, int PER_LANE>
cudaError_t launch_rows(const SharedArgs& p, cudaStream_t stream) {
    const long long blocks = ((long long)p.rows * p.nq + 3) / 4;
    return fr_launch(rows_kernel<T, PER_LANE>, dim3((unsigned)blocks, (unsigned)p.parts), dim3(128), 0, stream, p);
}

template <typename T>
int run(const SharedArgs& p, cudaStream_t stream) {
    FR_CUDA((p.hd <= 64 ? launch_rows<T, 2>(p, stream) : p.hd <= 128 ? launch_rows<T, 4>(p, stream) : launch_rows<T, 8>(p, stream)));
    FR_CHECK_LAUNCH("attention_shared");
    if (p.parts > 1) {
        const long long blocks = ((long long)p.rows * p.nq + 3) / 4;
        FR_CUDA(fr_launch(merge_kernel<T>, dim3((unsigned)blocks), dim3(128), 0, stream, p));
        FR_CHECK_LAUNCH("attention_shared (merge)");
    }
    return FR_OK;
}

}  // namespace

// Working memory of a call, in floats.
FR_EXPORT long long attention_shared_floats(int rows, int n_seqs, int max_q_len, int max_kv_len, int prefix, int nq, int nkv, int hd,
                                            int window, int dtype) {
    if (rows <= 0 || nq <= 0 || hd <= 0) return 0;
    return floats_of(plan_of(rows, nq, max_kv_len, window), rows, nq, hd);
}

// How many kernels a call launches.
FR_EXPORT int attention_shared_launches(int rows, int n_seqs, int max_q_len, int max_kv_len, int prefix, int nq, int nkv, int hd,
                                        int window, int dtype) {
    if (rows <= 0 || nq <= 0 || hd <= 0) return 0;
    return plan_of(rows, nq, max_kv_len, window).parts > 1 ? 2 : 1;
}

// seq_start, seq_qlen: per sequence its first row and its rows in this step.  max_kv_len: a bound on every row's position + 1, which
// only shares the work out.  scratch: attention_shared_floats floats.
FR_EXPORT int attention_shared(const void* q, long long q_stride, void* out, const void* k_pool, const void* v_pool, int pool_pages, int page,
                               const int* prefix_table, int prefix, const int* block_table, int n_seqs, int table_width, const int* row_seq,
                               const int* row_pos, const int* seq_start, const int* seq_qlen, int rows, int max_q_len, int max_kv_len,
                               int nq, int nkv, int hd, int window, float scale, float* scratch, long long scratch_floats, int* status,
                               int dtype, cudaStream_t stream) {
    if (rows <= 0 || n_seqs <= 0) return FR_OK;
    if (dtype != FR_F32 && dtype != FR_BF16) FR_REFUSE("attention_shared: unknown dtype %d", dtype);
    if (nq < 1 || nkv < 1 || nq % nkv || hd < 1 || hd > MOST_HEAD)
        FR_REFUSE("attention_shared: %d heads on %d kv heads of %d numbers (at most %d)", nq, nkv, hd, MOST_HEAD);
    if (prefix < 0 || page < 1 || pool_pages < 1 || table_width < 0 || window < 0)
        FR_REFUSE("attention_shared: prefix %d, pages of %d, %d of them, a table %d wide, window %d", prefix, page, pool_pages, table_width, window);
    if (!(scale > 0.f) || !(scale < INFINITY)) FR_REFUSE("attention_shared: a scale of %g", (double)scale);
    const Plan plan = plan_of(rows, nq, max_kv_len, window);
    if (scratch_floats < floats_of(plan, rows, nq, hd)) FR_REFUSE("attention_shared: %lld floats of working memory are too few", scratch_floats);
    SharedArgs p = {};
    p.q = q; p.out = out; p.k_pool = k_pool; p.v_pool = v_pool; p.prefix_table = prefix_table; p.block_table = block_table;
    p.row_seq = row_seq; p.row_pos = row_pos; p.q_stride = q_stride; p.rows = rows; p.n_seqs = n_seqs; p.nq = nq; p.nkv = nkv; p.hd = hd;
    p.window = window; p.prefix = prefix; p.page = page; p.pool_pages = pool_pages; p.table_width = table_width; p.parts = plan.parts;
    p.part = scratch; p.stat = scratch + (long long)rows * nq * plan.parts * hd;
    p.scale_log2 = scale * 1.4426950408889634f;
    return dtype == FR_F32 ? run<float>(p, stream) : run<bf16>(p, stream);
}
