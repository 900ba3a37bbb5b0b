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
#include <cuda.h>
#include <math.h>

#include <string.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "divide.cuh"
#include "tc_common.cuh"

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
    // the tensor-core kernel's
    const int* seq_start;     // [n_seqs] first row of each sequence, its rows in this step
    const int* seq_qlen;
    int* status;
    int whole;                // 1: a CTA walks prefix and own keys of one sequence's rows; 0: CTAs of one or the other, parts joined
    int jobs, prefix_jobs, prefix_splits, own_splits;           // prefix_splits 0: parts are not of one range or the other
    int covered;              // rows of a sequence that the grid's own tiles reach
    int tiles, own_tiles, tile_tokens;                // row tiles of the prefix' jobs and of a sequence; token rows of a tile
    // (a CTA's begin is a chain of latencies, of which a dozen divisions by numbers that only the host knows were 0.8 us)
    FrDivide by_tiles, by_kv, by_seqs, by_inner, by_group, by_heads, by_pieces, by_prefix_splits, by_own_splits;
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
// A block per (row, head): as many parts at a time as its threads make of a head's pieces (of VEC numbers), the first four of each
// thread fetched beside the statistics.  A part that saw no key has l = 0 and drops out; what its o holds does not count.  (One warp
// that took part after part waited for memory once for each: 16 rows x 28 heads x 75 parts of 128 in 45 us.)
template <typename T, int VEC>
__global__ void __launch_bounds__(VEC == 4 ? 128 : 256) merge_kernel(const SharedArgs p) {
    constexpr int THREADS = VEC == 4 ? 128 : 256, AHEAD = 4;
    __shared__ float weight[MOST_PARTS];
    __shared__ float inv_sum;
    __shared__ float partial[THREADS * VEC];
    fr_pdl_wait();
    fr_pdl_launch();
    const int tid = threadIdx.x, lane = tid & 31;
    const long long item = blockIdx.x;
    const int row = p.by_heads((int)blockIdx.x);
    const int pieces = p.hd / VEC, at_once = p.by_pieces(THREADS), sub = p.by_pieces(tid), piece = tid - sub * pieces;
    const bool busy = sub < at_once;
    const float* from = p.part + (size_t)item * p.parts * p.hd + piece * VEC;
    float v[AHEAD][VEC];
    auto fetch = [&](int s, float (&to)[VEC]) {
        if (busy && s < p.parts) {
            if (VEC == 4) *(float4*)to = *(const float4*)(from + (size_t)s * p.hd);
            else to[0] = from[(size_t)s * p.hd];
        }
    };
    // lane s has the statistics of parts s and s + 32
    float2 ml[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
    if (tid < 32) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (lane + 32 * i < p.parts) ml[i] = *(const float2*)(p.stat + 2 * ((size_t)item * p.parts + lane + 32 * i));
    }
    const int seq = p.row_seq[row];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(sub + i * at_once, v[i]);
    if (seq < 0 || seq >= p.n_seqs) return;
    if (tid < 32) {
        // own parts are there for rows that the sequence's range names
        int parts = p.parts;
        if (p.prefix_splits > 0) {
            const int t = row - p.seq_start[seq];
            if (t < 0 || t >= min(p.seq_qlen[seq], p.covered)) parts = p.prefix_splits;
        }
        float m[2], l[2], f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] = lane + 32 * i < parts ? ml[i].y : 0.f;
            m[i] = l[i] == 0.f ? -INFINITY : ml[i].x;
        }
        const float big = fr_warp_max(fmaxf(m[0], m[1]));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            f[i] = l[i] == 0.f ? 0.f : exp2f(m[i] - big);
            weight[lane + 32 * i] = f[i];
        }
        const float sum = fr_warp_sum(f[0] * l[0] + f[1] * l[1]);
        if (lane == 0) inv_sum = sum > 0.f ? 1.f / sum : sum;        // (0: nothing seen; a NaN stays one)
    }
    __syncthreads();
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
    for (int s0 = sub; s0 < p.parts; s0 += AHEAD * at_once) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + i * at_once;
            const float w = busy && s < p.parts ? weight[s] : 0.f;
            if (w != 0.f)
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] = fmaf(w, v[i][j], acc[j]);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch(s0 + (AHEAD + i) * at_once, v[i]);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) partial[tid * VEC + j] = acc[j];
    __syncthreads();
    // (in the order of the parts' residues, whatever the number of threads: the same bits every time)
    for (int d = tid; d < p.hd; d += THREADS) {
        float sum = 0.f;
        for (int i = 0; i < at_once; ++i) sum += partial[i * p.hd + d];
        fr_store((T*)p.out + (size_t)item * p.hd + d, sum * inv_sum);
    }
}

// ------------------------------------------------------------------ jobs of tiles
// Both kernels below work on tiles: the group heads of consecutive token rows, for one kv head.  For the prefix a tile's token rows are
// any consecutive rows of the step, whatever sequences they belong to: that is what reads the prefix once for all.  For own keys they
// are rows of one sequence.  A CTA has one tile and one of three jobs:
//
//   prefix   consecutive rows of the step, a share of the prefix' blocks of keys    -> a part
//   own      rows of one sequence, a share of its own blocks                        -> a part
//   whole    rows of one sequence, all of the prefix' blocks and then its own       -> the result (many rows per sequence)

// the last position that a row at `pos` sees: its own, no further than the tables have room; -1: it sees nothing.  (Its window ends at
// its own position, wherever the tables end: the first position that it sees goes by `pos`, and may lie behind the last.)
__device__ __forceinline__ int last_seen(const SharedArgs& p, int pos) {
    const long long room = (long long)p.prefix + (long long)p.table_width * p.page;
    return max(-1, (int)min((long long)pos, room - 1));
}

// Keys [lo, hi] of a range of pages that the CTA's rows see between them (none: hi < lo), block `first` its first one here, n blocks.
struct Range {
    int lo, hi, first, n;
};
struct Job {
    int kvh, seq, row0, n_tok, part;      // n_tok token rows from row0 on
    Range seg0, seg1;                     // of the prefix; of own keys, numbered from the prefix' end
    int all_lo, all_hi;                   // positions that every row sees that sees any; in between them others may see more
    bool uneven;                          // there are positions that some rows see and others do not, or none between the rows' windows
    bool early;
    int first_page;                       // of own keys, looked up while the rows' positions are on the way (-2: not looked up)
};

// The sequences by their last position, greatest first (ties: the lower number first): own jobs are taken longest first.
__device__ __forceinline__ void order_by_length(const SharedArgs& p, int* s_order, int* s_last) {
    int last = -1;
    const int s = threadIdx.x;
    if (s < p.n_seqs) {
        const int begin = p.seq_start[s], count = p.seq_qlen[s];
        if (count > 0 && begin >= 0 && begin + (long long)count <= p.rows) last = p.row_pos[begin + count - 1];
        s_last[s] = last;
    }
    __syncthreads();
    if (s < p.n_seqs) {
        int before = 0;
        for (int other = 0; other < p.n_seqs; ++other) {
            const int theirs = s_last[other];
            before += theirs > last || (theirs == last && other < s) ? 1 : 0;
        }
        s_order[before] = s;
    }
    __syncthreads();
}

// Job number `index` of p.jobs.  Tiles of one kv head and share of the prefix are neighbours: they read the same pages at about the same
// time.  The prefix' shares (the most work) come first, a whole job's late rows first.  T token rows make a tile; s_pos: two numbers in
// shared memory, (INT_MAX, -1) behind a barrier; s_order: the sequences in the order in which they are taken (null: their own).  For all
// threads of the block.  early: a share of the prefix without a window does not wait for the rows' positions; its range then ends with
// the prefix, wherever the last of its rows is.
template <int keys, int threads>
__device__ __forceinline__ Job job_of(const SharedArgs& p, int index, int T, int* s_pos, const int* s_order, bool early) {
    Job job;
    job.first_page = -2;
    const bool prefix_job = !p.whole && index < p.prefix_jobs;
    int share, tile;
    if (prefix_job) {
        const int q = p.by_tiles(index);
        tile = index - q * p.tiles;
        share = p.by_kv(q);
        job.kvh = q - share * p.nkv;
        job.seq = 0;
        job.row0 = tile * T;
        job.part = share;
        job.n_tok = min(T, p.rows - job.row0);
    } else {
        // (whole: the sequences' tiles of one rank together; else the shares and kv heads of a sequence)
        const int x = index - p.prefix_jobs;
        int s;
        if (p.whole) {
            const int q = p.by_seqs(x);
            s = x - q * p.n_seqs;
            tile = p.by_kv(q);
            job.kvh = q - tile * p.nkv;
            share = 0;
        } else {
            const int q = p.by_inner(x), rest = x - q * (int)p.by_inner.by;
            tile = p.by_seqs(q);
            s = q - tile * p.n_seqs;
            share = p.by_kv(rest);
            job.kvh = rest - share * p.nkv;
        }
        job.seq = s_order != nullptr ? s_order[s] : s;
        job.part = p.prefix_splits + share;
        // (without a window the first share begins with the first page)
        if (!p.whole && share == 0 && p.window == 0 && p.table_width > 0) job.first_page = p.block_table[(size_t)job.seq * p.table_width];
        const int t0 = (p.own_tiles - 1 - tile) * T;
        const int begin = p.seq_start[job.seq], count = begin < 0 || begin > p.rows ? 0 : min(p.seq_qlen[job.seq], p.rows - begin);
        job.row0 = begin + t0;
        job.n_tok = max(0, min(T, count - t0));
    }
    job.seg0 = job.seg1 = Range{0, -1, 0, 0};
    job.early = early && prefix_job && p.window == 0;
    job.all_lo = job.all_hi = 0;
    job.uneven = false;
    if (job.early) {
        job.seg0.hi = p.prefix - 1;
    } else {
        int least = 0x7fffffff, most = -1;                         // of the rows' positions
        if (job.n_tok == 1) {                                      // (a one-token step: every thread looks for itself)
            const int of = p.row_seq[job.row0], pos = p.row_pos[job.row0];
            if (of >= 0 && of < p.n_seqs && pos >= 0) least = most = pos;
        } else {
            for (int t = threadIdx.x; t < job.n_tok; t += threads) {
                const int of = p.row_seq[job.row0 + t], pos = p.row_pos[job.row0 + t];
                if (of >= 0 && of < p.n_seqs && pos >= 0) {
                    atomicMin(&s_pos[0], pos);
                    atomicMax(&s_pos[1], pos);
                }
            }
            __syncthreads();
            least = s_pos[0];
            most = s_pos[1];
        }
        const int lo = most < 0 ? 0 : fr_first_key(least, p.window, 0), hi = last_seen(p, most);
        job.seg0.lo = lo;
        job.seg1.lo = max(0, lo - p.prefix);
        if (p.whole || prefix_job) job.seg0.hi = min(hi, p.prefix - 1);
        if (!prefix_job) job.seg1.hi = hi - p.prefix;
        job.all_lo = fr_first_key(most, p.window, 0);
        job.all_hi = last_seen(p, least);
        job.uneven = most >= 0 && (lo < job.all_lo || job.all_hi < hi);
    }
    // equal shares of the blocks, the first ones a block longer where they do not come out even
    const FrDivide& shares = prefix_job ? p.by_prefix_splits : p.by_own_splits;
    auto take_share = [&](Range& g) {
        if (g.hi < g.lo) return;
        const int first = g.lo / keys, n = g.hi / keys - first + 1;
        const int each = shares(n), more = n - each * (int)shares.by;
        g.first = first + share * each + min(share, more);
        g.n = each + (share < more ? 1 : 0);
    };
    take_share(job.seg0);
    take_share(job.seg1);
    return job;
}

// ------------------------------------------------------------------ float32 in tiles
// A block of 128 threads has 16 RPT rows and walks 32 keys at a time, which pass through shared memory once for all of them (two or
// four stages, 16-byte asynchronous copies; what no row of the block sees, and pages that a table leaves out, come as zeros; the page
// of a block is looked up a block before its copies are issued).  A thread has
// the scores of up to RPT rows (4 of a warp side by side, 16 apart) with four keys, then the same rows' results in HD / 8 channels, so
// that a row's scores, maximum and weights stay within a warp.  Bound by what shared memory reads where rows are many; a tile of few
// rows (one token's group heads) only takes the 16-row steps that it has.  43 rows of 5 sequences behind 1,773 keys, 16 heads on 2 of
// 112: 40 us (66 with 4 x 4 scores per thread); 16 rows behind 4,000 keys, 28 heads on 4 of 128: 51 (81).
namespace f32 {

constexpr int KEYS = 32, THREADS = 128, LS = KEYS + 8;
template <int HD>
constexpr int stages() { return HD > 64 ? 2 : 4; }
template <int HD, int RPT>
constexpr int smem_bytes() { return (16 * RPT * (HD + 4) + stages<HD>() * KEYS * (2 * HD + 4) + 16 * RPT * LS) * 4; }

template <int HD, int RPT>
__global__ void __launch_bounds__(THREADS) tiles_kernel(const SharedArgs p) {
    constexpr int ROWS = 16 * RPT, LQ = HD + 4, CH = HD / 32, STAGES = stages<HD>();      // CH: groups of four channels per thread
    extern __shared__ __align__(16) float tile_smem[];
    float* const sq = tile_smem;                                       // [ROWS][LQ]
    float* const sk = sq + ROWS * LQ;                                  // [STAGES][KEYS][LQ]
    float* const sv = sk + STAGES * KEYS * LQ;                         // [STAGES][KEYS][HD]
    float* const sp = sv + STAGES * KEYS * HD;                         // [ROWS][LS]
    __shared__ int s_pos[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, ty = lane >> 3, tx = lane & 7;
    if (tid == 0) {
        s_pos[0] = 0x7fffffff;
        s_pos[1] = -1;
    }
    __syncthreads();
    fr_pdl_wait();
    fr_pdl_launch();
    const int G = (int)p.by_group.by, T = p.tile_tokens;
    const Job job = job_of<KEYS, THREADS>(p, (int)blockIdx.x, T, s_pos, nullptr, false);
    const int n_rows = job.n_tok * G, n_blocks = job.seg0.n + job.seg1.n;
    auto range_of = [&](int i, int& j0, bool& own) {
        own = i >= job.seg0.n;
        j0 = (own ? job.seg1.first + i - job.seg0.n : job.seg0.first + i) * KEYS;
        return own ? job.seg1 : job.seg0;
    };
    // (pages that are whole blocks: all keys of a block lie in one)
    const bool one_page = p.page % KEYS == 0;
    auto page_of = [&](int i) {
        if (!one_page || i >= n_blocks) return -1;
        int j0;
        bool own;
        range_of(i, j0, own);
        return own ? p.block_table[(size_t)job.seq * p.table_width + j0 / p.page] : p.prefix_table[j0 / p.page];
    };
    auto fetch = [&](int i, int page) {
        if (i < n_blocks) {
            int j0;
            bool own;
            const Range g = range_of(i, j0, own);
            float* dk = sk + i % STAGES * KEYS * LQ;
            float* dv = sv + i % STAGES * KEYS * HD;
            const long long base = page >= 0 && page < p.pool_pages ? (long long)page * p.page + j0 % p.page : -1;
#pragma unroll
            for (int it = 0; it < KEYS * (HD / 4) / THREADS; ++it) {
                const int idx = tid + it * THREADS, key = idx / (HD / 4), c = idx % (HD / 4) * 4, j = j0 + key;
                long long at = -1;
                if (j >= g.lo && j <= g.hi && c < p.hd) at = !one_page ? place_of(p, job.seq, own ? j + p.prefix : j) : base >= 0 ? base + key : -1;
                const size_t from = at >= 0 ? ((size_t)at * p.nkv + job.kvh) * p.hd + c : 0;
                const int bytes = at >= 0 ? 16 : 0;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dk + key * LQ + c)),
                             "l"((const float*)p.k_pool + from), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dv + key * HD + c)),
                             "l"((const float*)p.v_pool + from), "r"(bytes) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int ahead[STAGES - 1];
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) ahead[i] = page_of(i);
    int next_page = page_of(STAGES - 1);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i, ahead[i]);
    for (int idx = tid; idx < ROWS * (HD / 4); idx += THREADS) {
        const int r = idx / (HD / 4), c = idx % (HD / 4) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        const int t = p.by_group(r);
        if (r < n_rows && c < p.hd) v = *(const float4*)((const float*)p.q + (size_t)(job.row0 + t) * p.q_stride + (size_t)(job.kvh * G + r - t * G) * p.hd + c);
        v.x *= p.scale_log2; v.y *= p.scale_log2; v.z *= p.scale_log2; v.w *= p.scale_log2;
        *(float4*)(sq + r * LQ + c) = v;
    }
    const int r0 = 4 * warp + ty;                                      // this thread's rows: r0 + 16 i
    int pos[RPT], first[RPT];
    bool live[RPT];
    float m[RPT], l[RPT], acc[RPT][4 * CH];
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
        const int r = r0 + 16 * i;
        live[i] = r < n_rows;
        pos[i] = -1;
        first[i] = 0;
        if (live[i]) {
            const int row = job.row0 + p.by_group(r), of = p.row_seq[row];
            live[i] = of >= 0 && of < p.n_seqs;
            if (live[i]) {
                first[i] = fr_first_key(p.row_pos[row], p.window, 0);
                pos[i] = last_seen(p, p.row_pos[row]);
            }
        }
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < 4 * CH; ++c) acc[i][c] = 0.f;
    }
    // one block of keys for the thread's first N rows
    auto work = [&](auto number, int i) {
        constexpr int N = decltype(number)::value;
        int j0;
        bool own;
        range_of(i, j0, own);
        // Four lanes (two of ty, two of tx) make the scores of all their rows with all their keys, each over every fourth group of four
        // dimensions; then each gets the sums that are its own.  Shared memory gives a warp 128 bytes a cycle, so 8 rows x 8 keys
        // per lane take as long to read as to multiply, where 4 x 4 take twice that: 11,800 -> 3,800 cycles a block of 128 dimensions.
        float part[2 * N][8];
#pragma unroll
        for (int a = 0; a < 2 * N; ++a)
#pragma unroll
            for (int b = 0; b < 8; ++b) part[a][b] = 0.f;
        const int quarter = (ty & 1) * 2 + (tx & 1);
        const float* q0 = sq + (4 * warp + (ty & 2)) * LQ + 4 * quarter;
        const float* k0 = sk + i % STAGES * KEYS * LQ + (tx & 6) * LQ + 4 * quarter;
#pragma unroll 1
        for (int d = 0; d < HD; d += 16) {
            float4 q[2 * N];
#pragma unroll
            for (int a = 0; a < 2 * N; ++a) q[a] = *(const float4*)(q0 + (16 * (a >> 1) + (a & 1)) * LQ + d);
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const float4 k = *(const float4*)(k0 + (8 * (b >> 1) + (b & 1)) * LQ + d);
#pragma unroll
                for (int a = 0; a < 2 * N; ++a) part[a][b] = fmaf(q[a].x, k.x, part[a][b]);
#pragma unroll
                for (int a = 0; a < 2 * N; ++a) part[a][b] = fmaf(q[a].y, k.y, part[a][b]);
#pragma unroll
                for (int a = 0; a < 2 * N; ++a) part[a][b] = fmaf(q[a].z, k.z, part[a][b]);
#pragma unroll
                for (int a = 0; a < 2 * N; ++a) part[a][b] = fmaf(q[a].w, k.w, part[a][b]);
            }
        }
        float s[N][4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float half[2 * N];
#pragma unroll
            for (int a = 0; a < 2 * N; ++a) {
                const float mine = tx & 1 ? part[a][2 * b + 1] : part[a][2 * b], other = tx & 1 ? part[a][2 * b] : part[a][2 * b + 1];
                half[a] = mine + __shfl_xor_sync(0xffffffffu, other, 1);
            }
#pragma unroll
            for (int a = 0; a < N; ++a) {
                const float mine = ty & 1 ? half[2 * a + 1] : half[2 * a], other = ty & 1 ? half[2 * a] : half[2 * a + 1];
                s[a][b] = mine + __shfl_xor_sync(0xffffffffu, other, 8);
            }
        }
#pragma unroll
        for (int a = 0; a < N; ++a) {
            // columns hi < column or column < lo are masked
            const int hi = (own ? pos[a] - p.prefix : min(pos[a], p.prefix - 1)) - j0, lo = first[a] - (own ? p.prefix : 0) - j0;
            float big = m[a];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int key = tx + 8 * b;
                if (key > hi || key < lo) s[a][b] = -INFINITY;
                big = fmaxf(big, s[a][b]);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const float ref = big == -INFINITY ? 0.f : big;            // (nothing seen yet: weights against 0, all of them 0)
            const float keep = exp2f(m[a] - ref);
            float sum = 0.f;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const float w = exp2f(s[a][b] - ref);
                sum += w;
                sp[(r0 + 16 * a) * LS + tx + 8 * b] = w;
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l[a] = l[a] * keep + sum;
            m[a] = big;
#pragma unroll
            for (int c = 0; c < 4 * CH; ++c) acc[a][c] *= keep;
        }
        __syncwarp();
        const float* v0 = sv + i % STAGES * KEYS * HD + 4 * tx;
        auto results = [&](auto choosy) {
#pragma unroll 2
            for (int j = 0; j < KEYS; j += 4) {
                float w[N][4];
#pragma unroll
                for (int a = 0; a < N; ++a) *(float4*)w[a] = *(const float4*)(sp + (r0 + 16 * a) * LS + j);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        const float4 v = *(const float4*)(v0 + (j + e) * HD + 32 * c);
#pragma unroll
                        for (int a = 0; a < N; ++a) {
                            if (decltype(choosy)::value && w[a][e] == 0.f) continue;
                            acc[a][4 * c] = fmaf(w[a][e], v.x, acc[a][4 * c]);
                            acc[a][4 * c + 1] = fmaf(w[a][e], v.y, acc[a][4 * c + 1]);
                            acc[a][4 * c + 2] = fmaf(w[a][e], v.z, acc[a][4 * c + 2]);
                            acc[a][4 * c + 3] = fmaf(w[a][e], v.w, acc[a][4 * c + 3]);
                        }
                    }
            }
        };
        // (where some rows see positions that others do not: a value that a row does not see may be anything, and zero times infinity is
        // not zero)
        const Range& g = own ? job.seg1 : job.seg0;
        const int seen_from = max(j0, g.lo) + (own ? p.prefix : 0), seen_to = min(j0 + KEYS - 1, g.hi) + (own ? p.prefix : 0);
        if (job.uneven && (seen_from < job.all_lo || seen_to > job.all_hi)) results(std::true_type{});
        else results(std::false_type{});
        __syncwarp();
    };
    const int steps = (n_rows - 4 * warp + 15) / 16;                   // 16-row steps in which this warp has rows
    for (int i = 0; i < n_blocks; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncthreads();                                               // this block of keys is here, and everyone is done with the one before
        fetch(i + STAGES - 1, next_page);
        next_page = page_of(i + STAGES);
        if (steps <= 0) continue;
        if (RPT >= 2 && steps > RPT / 2) work(std::integral_constant<int, RPT>{}, i);
        else if (RPT >= 4 && steps > RPT / 4) work(std::integral_constant<int, (RPT >= 2 ? RPT / 2 : 1)>{}, i);
        else work(std::integral_constant<int, (RPT >= 4 ? RPT / 4 : 1)>{}, i);
    }
#pragma unroll
    for (int a = 0; a < RPT; ++a) {
        if (!live[a]) continue;
        const int r = r0 + 16 * a, t = p.by_group(r);
        const size_t item = (size_t)(job.row0 + t) * p.nq + (size_t)job.kvh * G + r - t * G, at = item * p.parts + job.part;
        const float inv = l[a] > 0.f ? 1.f / l[a] : l[a];              // (a NaN stays one)
        if (p.whole && l[a] == 0.f)                                    // nothing seen: 0, whatever was multiplied by 0
#pragma unroll
            for (int c = 0; c < 4 * CH; ++c) acc[a][c] = 0.f;
        float* to = p.whole ? (float*)p.out + item * p.hd : p.part + at * p.hd;
        if (!p.whole && tx == 0) *(float2*)(p.stat + 2 * at) = make_float2(m[a], l[a]);
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (4 * tx + 32 * c < p.hd)
                *(float4*)(to + 4 * tx + 32 * c) = p.whole ? make_float4(acc[a][4 * c] * inv, acc[a][4 * c + 1] * inv, acc[a][4 * c + 2] * inv, acc[a][4 * c + 3] * inv)
                                                           : make_float4(acc[a][4 * c], acc[a][4 * c + 1], acc[a][4 * c + 2], acc[a][4 * c + 3]);
    }
}

template <int HD, int RPT>
int launch(const SharedArgs& p, long long ctas, cudaStream_t stream) {
    static std::atomic<unsigned long long> configured{0};             // a bit per device
    int device = 0;
    FR_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if (!(configured.load() & bit)) {
        FR_CUDA(cudaFuncSetAttribute(tiles_kernel<HD, RPT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<HD, RPT>()));
        configured.fetch_or(bit);
    }
    FR_CUDA(fr_launch(tiles_kernel<HD, RPT>, dim3((unsigned)ctas), dim3(THREADS), (size_t)smem_bytes<HD, RPT>(), stream, p));
    FR_CHECK_LAUNCH("attention_shared (float32 tiles)");
    return FR_OK;
}

template <int HD>
int launch_rows(const SharedArgs& p, int tile_rows, long long ctas, cudaStream_t stream) {
    return tile_rows == 64 ? launch<HD, 4>(p, ctas, stream) : tile_rows == 32 ? launch<HD, 2>(p, ctas, stream) : launch<HD, 1>(p, ctas, stream);
}

}  // namespace f32

// ------------------------------------------------------------------ bf16 on the tensor cores
// Both products are tcgen05.mma with scores, weights and results in tensor memory.  A tile is 128 rows of one kv head; row r of it
// stands for (token row r / G, group head r % G), G = heads / kv heads.
//
//   warp 0      TMA: the queries (a 4-d box [64 dims][G heads][1][T rows] per 64-dim slice lands as rows t * G + g, 128-byte
//               swizzle), then K of the block after and V of this one (a block of 64 keys is a page); a page that a table leaves out
//               is loaded from beyond the pool's last row, which fills zeros
//   warp 1      tensor memory; one lane issues S = Q K^T two blocks ahead of O += P V
//   warps 2-5   one thread per row: maximum, exponentials, running maximum and sum; P goes back into tensor memory (two bf16
//               numbers a weight) over its scores.  The reference maximum only moves when the true one has grown by more than 8 (in
//               log2 units; weights stay below 2^8); O is rescaled then.
//
// Scores, sums, weights and results are 32-bit in effect: P enters the second product as two bf16 numbers, the weight rounded over the
// first half of its scores' columns and what rounding left over the second half, each with the same values.  One number alone was off by
// as much again as the result's own rounding (norm of the error against 64 bits 0.0023 of the result's, 0.0017 with two), and which
// precision a caller got went by page size and alignment.  The second product takes twice its time for it: on one card 46 us for 41 (64
// one-token rows behind 16,001), 333 for 273 (the prompts).
//
// A CTA takes 101 KB of shared memory and half the tensor memory, so two share an SM and one's softmax runs beside the other's products.
// 16 prompts of 2,188 rows in all behind 8,000 keys, 28 heads on 4 of 128: 289 us, 0.82 PFLOP/s, and 336 in a run of seconds, whose
// power lowers the clock.  Of an SM's cycles for a block the first product's instructions take 8 x 48 (at 64 keys each reads twice as much
// of Q as of K) and the second's 2 x 4 x 64: the tensor core is busy for 72 of 100 cycles.
//
// What else was tried, with weights of one number, where the prompts took 238 us and 64 one-token rows behind 16,001 keys 37: two tiles
// and blocks of 128 keys in one CTA per SM (288 for 250, 71 for 52 then); a fourth of the exponentials as polynomials (no change); scores
// fetched at once so that one buffer serves, with half of Q in tensor memory (276 us); two threads per row (290); two groups of warps that
// take blocks in turn and hand the reference maximum over (392, 96 registers a thread); tiles of few rows on mma.sync, a block of keys per
// warp (1.13 us a block of one CTA for 0.68).  Where jobs are more than CTAs, the CTAs stay and take one job of every round, longest first
// (64 one-token rows 37 us; 48.5 with a CTA per job).
//
// A row's result depends on nothing that it does not see.  Weights there are 0, but zero times infinity is not: in blocks that all rows of
// the CTA see alike, values of positions that none sees are zeroed in shared memory before the product; in blocks where rows see different
// ranges (the last ones of a prompt's tile, the edges of windows, a prefix with rows inside it) all values that are not finite are taken
// out, and a row that sees one gets it at its end, for which those blocks' pages are read again (prompts 336 us for 333).  A row that gives
// a weight to a value that is not finite has no finite number there.
//
// Every wait on an mbarrier is bounded; a wait that gives up leaves a code in `status` and all roles leave their loops.
namespace tcore {

using namespace tc;

constexpr int ROWS = 128, PAGE = 64;
constexpr int SLICE = ROWS * 128;         // bytes of 128 rows of 64 numbers

constexpr int KEYS = 64, THREADS = 192;
constexpr int KSLICE = KEYS * 128, STAGE = 2 * KSLICE;        // a block's keys (or values): two slices of 64 dims
constexpr int TMEM = 256;                                     // columns: S of even blocks, S of odd blocks (P over each one's first half), O
constexpr int SMEM = 2 * SLICE + 4 * STAGE + 1024 + 256 + 2 * 4 * THREADS;      // (256: barriers and single words)

__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
                 : "memory");
}
// an operand whose contiguous dimension is N: 8 consecutive k form a 1024-byte swizzle atom of 64 n; sbo between atoms along k, lbo
// along n
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
        "%24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 2^x by the special-function unit alone (results below 2^-126 become 0)
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// the greatest of three; two sums, two multiply-adds in one instruction
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ unsigned long long two(float lo, float hi) {
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void halves(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
// two bf16 numbers: whether one is infinite or NaN; such ones replaced by zeros
__device__ __forceinline__ bool not_finite(uint32_t two_numbers) {
    return (two_numbers & 0x7f80u) == 0x7f80u || (two_numbers & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ uint32_t finite_of(uint32_t two_numbers) {
    return ((two_numbers & 0x7f80u) == 0x7f80u ? 0u : two_numbers & 0xffffu) | ((two_numbers & 0x7f800000u) == 0x7f800000u ? 0u : two_numbers & 0xffff0000u);
}
// D[tmem] (+)= A[tmem] * B[smem]: lane = row, two bf16 per column of A
__device__ __forceinline__ void mma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__global__ void __launch_bounds__(THREADS, 2)
tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const SharedArgs p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* s_q = smem;                              // [2 slices][128 rows][128 B]
    uint8_t* s_k = s_q + 2 * SLICE;                   // [2 stages][2 slices][KEYS][128 B]
    uint8_t* s_v = s_k + 2 * STAGE;
    uint64_t* bars = (uint64_t*)(s_v + 2 * STAGE);
    // bars: q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], pv_done[2]
    uint32_t* tmem_slot = (uint32_t*)(bars + 15);
    // a wait gave up; least, greatest position of a live row, for even and odd rounds; room for order_by_length; values were taken out, for
    // even and odd rounds
    int* s_pos = (int*)(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t q_full = smem_u32(bars), k_full = smem_u32(bars + 1), k_empty = smem_u32(bars + 3);
    const uint32_t v_full = smem_u32(bars + 5), v_empty = smem_u32(bars + 7);
    const uint32_t s_full = smem_u32(bars + 9), p_full = smem_u32(bars + 11), pv_done = smem_u32(bars + 13);

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int b = 0; b < 2; ++b) {
            mbar_init(k_full + 8 * b, 1);
            mbar_init(k_empty + 8 * b, 1);
            mbar_init(v_full + 8 * b, 1);
            mbar_init(v_empty + 8 * b, 1);
            mbar_init(s_full + 8 * b, 1);
            mbar_init(p_full + 8 * b, 128);
            mbar_init(pv_done + 8 * b, 1);
        }
        s_pos[0] = 0;
        s_pos[1] = s_pos[3] = 0x7fffffff;
        s_pos[2] = s_pos[4] = -1;
        s_pos[5 + 2 * THREADS] = s_pos[6 + 2 * THREADS] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    fr_pdl_wait();
    if (threadIdx.x == 0) fr_pdl_launch();

    const int G = (int)p.by_group.by, T = p.tile_tokens;
    const int slices = (p.hd + 63) / 64;
    int* s_order = nullptr;
    if (!p.whole && p.n_seqs <= THREADS && p.jobs > (int)gridDim.x) {
        s_order = s_pos + 5;
        order_by_length(p, s_order, s_order + THREADS);
    }
    // The CTA's jobs: one of every round of the grid, each round in the other direction than the one before, so that who had the
    // longest of a round has the shortest of the next.
    int blocks_before = 0, loads_before = 0;          // blocks and queries' tiles of the jobs so far: what the barriers' phases count
    for (int round = 0;; ++round) {
    const long long index = (long long)round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
    if ((long long)round * gridDim.x >= p.jobs) break;
    if (index >= p.jobs) continue;
    int* const s_range = s_pos + 1 + 2 * (round & 1);
    volatile int* const s_taken = s_pos + 5 + 2 * THREADS + (round & 1);
    const Job job = job_of<KEYS, THREADS>(p, (int)index, T, s_range, s_order, true);
    const Range seg0 = job.seg0, seg1 = job.seg1;
    const int kvh = job.kvh, seq = job.seq, row0 = job.row0, n_tok = job.n_tok, part = job.part;
    const int n_blocks = seg0.n + seg1.n, before = blocks_before;
    auto first_key_of = [&](int i) { return (i < seg0.n ? seg0.first + i : seg1.first + i - seg0.n) * KEYS; };
    auto last_key_of = [&](int i) { return i < seg0.n ? seg0.hi : seg1.hi; };
    // stage of block i, and the parity of that stage's use
    auto stage_of = [&](int i) { return (before + i) & 1; };
    auto parity_of = [&](int i) { return ((before + i) >> 1) & 1; };

    if (warp == 0) {
        if (n_blocks > 0 && elect_one()) {
            mbar_expect_tx(q_full, (uint32_t)(slices * 64 * G * T * 2));
            for (int s = 0; s < slices; ++s) load_4d(smem_u32(s_q + s * SLICE), &map_q, s * 64, 0, kvh, row0, q_full);
            auto load = [&](int i, const CUtensorMap* map, uint8_t* ring, uint32_t full, uint32_t empty) {
                const int b = stage_of(i), par = parity_of(i);
                if (!mbar_wait(empty + 8 * b, par ^ 1, p.status, 31)) return false;
                mbar_expect_tx(full + 8 * b, (uint32_t)(slices * KSLICE));
                const int* table = i < seg0.n ? p.prefix_table : p.block_table + (size_t)seq * p.table_width;
                int page = i == 0 && job.first_page != -2 ? job.first_page : table[first_key_of(i) / PAGE];
                if (page < 0 || page >= p.pool_pages) page = p.pool_pages;              // beyond the pool: zeros
                for (int s = 0; s < slices; ++s)
                    load_3d(smem_u32(ring) + (uint32_t)(b * STAGE + s * KSLICE), map, s * 64, kvh, page * PAGE, full + 8 * b);
                return true;
            };
            bool ok = load(0, &map_k, s_k, k_full, k_empty);
            for (int i = 0; i < n_blocks && ok; ++i) {
                if (i + 1 < n_blocks) ok = load(i + 1, &map_k, s_k, k_full, k_empty);
                if (ok) ok = load(i, &map_v, s_v, v_full, v_empty);
            }
            if (!ok) s_pos[0] = 1;
        }
    } else if (warp == 1) {
        if (n_blocks > 0 && elect_one()) {
            const uint32_t idesc_qk = instr_desc(ROWS, KEYS);
            const uint32_t idesc_pv = instr_desc(ROWS, p.hd) | (1u << 16);              // B is MN-major
            const int k_steps = p.hd / 16;
            bool ok = mbar_wait(q_full, loads_before & 1, p.status, 32);
            // (descriptors are made once and stepped: a lone thread issues all of this)
            const uint64_t dq0 = smem_desc(smem_u32(s_q)), dk0 = smem_desc(smem_u32(s_k)), dv0 = desc_mn(smem_u32(s_v), KSLICE, 1024);
            auto scores = [&](int i) {
                const int b = stage_of(i), par = parity_of(i);
                if (!mbar_wait(k_full + 8 * b, par, p.status, 33)) return false;
                tc_fence_after();
                uint64_t da = dq0, db = dk0 + (uint64_t)(b * (STAGE >> 4));
                const uint32_t d = tmem + KEYS * b;
                for (int ks = 0; ks < k_steps; ++ks) {
                    tc_mma(d, da, db, idesc_qk, ks > 0 ? 1u : 0u);
                    // 32 bytes on in the 128-byte row; after four of them the next slice of 64 dims
                    da += (ks & 3) == 3 ? (uint64_t)((SLICE >> 4) - 6) : 2ull;
                    db += (ks & 3) == 3 ? (uint64_t)((KSLICE >> 4) - 6) : 2ull;
                }
                tc_commit(s_full + 8 * b);
                tc_commit(k_empty + 8 * b);
                return true;
            };
            // The scores run two blocks ahead of the second product; the tensor core takes its instructions in order, so S of block i
            // may overwrite P of block i - 2.
            if (ok) ok = scores(0);
            if (ok && n_blocks > 1) ok = scores(1);
            for (int i = 0; i < n_blocks && ok; ++i) {
                const int b = stage_of(i), par = parity_of(i);
                if (!(ok = mbar_wait(v_full + 8 * b, par, p.status, 34))) break;
                if (!(ok = mbar_wait(p_full + 8 * b, par, p.status, 35))) break;
                tc_fence_after();
                const int steps = (min(KEYS, last_key_of(i) - first_key_of(i) + 1) + 15) / 16;
                uint64_t db = dv0 + (uint64_t)(b * (STAGE >> 4));
                uint32_t pa = tmem + KEYS * b, keep = i > 0 ? 1u : 0u;
                for (int ks = 0; ks < steps; ++ks) {
                    mma_ta(tmem + 2 * KEYS, pa, db, idesc_pv, keep);
                    mma_ta(tmem + 2 * KEYS, pa + KEYS / 2, db, idesc_pv, 1u);
                    keep = 1u;
                    pa += 8;                                   // 16 keys of P: 8 columns
                    db += (uint64_t)(16 * 128 >> 4);           // 16 keys of V
                }
                tc_commit(pv_done + 8 * b);
                tc_commit(v_empty + 8 * b);
                if (i + 2 < n_blocks) ok = scores(i + 2);
            }
            if (!ok) s_pos[0] = 1;
        }
    } else {
        const int quarter = warp & 3;                          // the tensor-memory lanes that this warp may touch: 32 * quarter ..
        const int r = quarter * 32 + lane, t = p.by_group(r), g = r - t * G;
        const int row = row0 + t;
        int pos = -1, first = 0;                               // the last and the first position that the row sees
        bool live = r < T * G && t < n_tok;
        if (live) {
            const int of = p.row_seq[row];
            live = of >= 0 && of < p.n_seqs;
            if (live) {
                first = fr_first_key(p.row_pos[row], p.window, 0);
                pos = last_seen(p, p.row_pos[row]);
            }
        }
        const bool any = __any_sync(0xffffffffu, live);        // a warp without rows only keeps the barriers going
        int prefix_hi = seg0.hi;                               // the last prefix position that a row of the CTA sees
        int all_lo = job.all_lo, all_hi = job.all_hi;
        bool uneven = job.uneven;
        if (job.early) {
            if (live && pos >= 0) {
                atomicMin(&s_range[0], pos);
                atomicMax(&s_range[1], pos);
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            prefix_hi = min(seg0.hi, s_range[1]);
            all_lo = 0;
            all_hi = s_range[0];
            uneven = all_hi < prefix_hi;
        }
        // Whether some row sees a position of block i that another does not: of each range the blocks but [from, to) are mixed.
        int even_from0 = 0, even_to0 = seg0.n, even_from1 = seg0.n, even_to1 = n_blocks;
        if (uneven) {
            const int lo0 = all_lo, hi0 = all_hi, lo1 = all_lo - p.prefix, hi1 = all_hi - p.prefix;          // in each range's numbers
            if (seg0.lo < lo0) even_from0 = (int)(((unsigned)lo0 + KEYS - 1) / KEYS) - seg0.first;
            if (prefix_hi > hi0) even_to0 = max(hi0 + 1, 0) / KEYS - seg0.first;
            if (seg1.lo < lo1) even_from1 = seg0.n + (int)(((unsigned)lo1 + KEYS - 1) / KEYS) - seg1.first;
            if (seg1.hi > hi1) even_to1 = seg0.n + max(hi1 + 1, 0) / KEYS - seg1.first;
        }
        auto mixed = [&](int i) { return i < seg0.n ? i < even_from0 || i >= even_to0 : i < even_from1 || i >= even_to1; };
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16, t_o = tmem + lane_addr + 2 * KEYS;
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        for (int i = 0; i < n_blocks; ++i) {
            const int b = stage_of(i), par = parity_of(i);
            const bool own = i >= seg0.n;
            const int j0 = first_key_of(i);
            if (!(ok = mbar_wait(s_full + 8 * b, par, p.status, 36))) break;
            tc_fence_after();
            const uint32_t t_s = tmem + lane_addr + KEYS * b;
            if (any) {
                uint32_t raw[KEYS];
                ld32(t_s, &raw[0]);
                ld32(t_s + 32, &raw[32]);
                tc_ld_wait();
                // columns hi < j or j < lo are masked; most blocks need no mask for any of the warp's rows
                const int hi = (own ? pos - p.prefix : min(pos, p.prefix - 1)) - j0, lo = first - (own ? p.prefix : 0) - j0;
                if (__any_sync(0xffffffffu, live && (hi < KEYS - 1 || lo > 0))) {
#pragma unroll
                    for (int j = 0; j < KEYS; ++j)
                        if (j > hi || j < lo) raw[j] = 0xff800000u;      // -inf
                }
                // (the maximum in four strands; the positive scale is applied to the result)
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < KEYS; j += 2) mx4[(j >> 1) & 3] = max3(mx4[(j >> 1) & 3], __uint_as_float(raw[j]), __uint_as_float(raw[j + 1]));
                const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]) * p.scale_log2;
                const bool grow = mx > m_run + 8.f;
                if (__any_sync(0xffffffffu, grow)) {
                    const float alpha = grow ? exp2f(m_run - mx) : 1.f;      // 0 for a row that had seen no key
                    if (grow) {
                        m_run = mx;
                        l_run *= alpha;
                    }
                    if (i > 0) {
                        // Every product into O so far must be done: that of block i - 2 is (this block's scores were issued behind
                        // it), so the wait for the other stage's phase is unambiguous.
                        if (!(ok = mbar_wait(pv_done + 8 * (b ^ 1), parity_of(i - 1), p.status, 38))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < p.hd; c += 16) {
                            uint32_t o16[16];
                            tc_ld16(t_o + c, o16);
                            tc_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o16[j] = __float_as_uint(__uint_as_float(o16[j]) * alpha);
                            st16(t_o + c, o16);
                        }
                        st_wait();
                    }
                }
                // a masked score is -inf and stays so; a row that has seen no key takes its exponentials against 0
                const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
                const unsigned long long scale2 = two(p.scale_log2, p.scale_log2), neg2 = two(neg_m, neg_m);
                unsigned long long sum2[2] = {0ull, 0ull};
#pragma unroll
                for (int h = 0; h < 2; ++h) {                  // (a half is on its way while the other is made)
                    uint32_t head[16], rest[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float x0, x1;
                        halves(fma2(two(__uint_as_float(raw[32 * h + j]), __uint_as_float(raw[32 * h + j + 1])), scale2, neg2), x0, x1);
                        const float e0 = exp2_fast(x0), e1 = exp2_fast(x1);
                        sum2[(j >> 1) & 1] = add2(sum2[(j >> 1) & 1], two(e0, e1));
                        // a weight is two bf16 numbers: itself rounded, and what rounding left (its last 2^-16 is lost)
                        const uint32_t w = pack2(e0, e1);
                        float r0, r1;
                        halves(fma2(two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)), two(-1.f, -1.f), two(e0, e1)), r0, r1);
                        head[j >> 1] = w;
                        rest[j >> 1] = pack2(r0, r1);
                    }
                    st16(t_s + 16 * h, head);
                    st16(t_s + KEYS / 2 + 16 * h, rest);
                }
                float sum4[4];
                halves(sum2[0], sum4[0], sum4[1]);
                halves(sum2[1], sum4[2], sum4[3]);
                l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
                st_wait();
            }
            const int in_lo = (own ? seg1.lo : seg0.lo) - j0, in_hi = (own ? seg1.hi : prefix_hi) - j0;
            if (mixed(i)) {
                // Values that are not finite are taken out (zero times infinity is not zero); rows that see them get them at the end.
                if (!(ok = mbar_wait(v_full + 8 * b, par, p.status, 37))) break;
                const int key = r & (KEYS - 1);
                bool found = false;
                for (int s = 0; s < slices; ++s) {
                    // (a row's eight pieces of 16 bytes shared by two threads, lanes in different banks)
                    uint32_t* line = (uint32_t*)(s_v + b * STAGE + s * KSLICE + key * 128);
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint4* const at = (uint4*)line + ((r + (r / KEYS) * 4 + q) & 7);
                        const uint4 v = *at;
                        if (not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w)) {
                            found |= key >= in_lo && key <= in_hi;             // (behind the last row's position nobody asks for them)
                            *at = make_uint4(finite_of(v.x), finite_of(v.y), finite_of(v.z), finite_of(v.w));
                        }
                    }
                }
                if (found) *s_taken = 1;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            } else if (in_lo > 0 || in_hi < KEYS - 1) {
                // positions that no row of the CTA sees: their values may be anything
                if (!(ok = mbar_wait(v_full + 8 * b, par, p.status, 37))) break;
                if (r < KEYS && (r < in_lo || r > in_hi)) {
                    for (int s = 0; s < slices; ++s) {
                        uint4* line = (uint4*)(s_v + b * STAGE + s * KSLICE + r * 128);
#pragma unroll
                        for (int q = 0; q < 8; ++q) line[q] = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            tc_fence_before();
            mbar_arrive(p_full + 8 * b);
        }
        if (ok && n_blocks > 0) {
            ok = mbar_wait(pv_done + 8 * stage_of(n_blocks - 1), parity_of(n_blocks - 1), p.status, 38);
            tc_fence_after();
        }
        if (!ok) s_pos[0] = 1;
        if (uneven) asm volatile("bar.sync 1, 128;" ::: "memory");          // (s_taken is everyone's)
        const bool taken = uneven && *s_taken != 0;
        if (ok && any) {
            const size_t item = (size_t)row * p.nq + (size_t)kvh * G + g;
            const bool seen = l_run != 0.f;                    // (a NaN is seen)
            const float inv = l_run > 0.f ? 1.f / l_run : l_run;
            const size_t at = item * p.parts + part;
            if (!p.whole && live) *(float2*)(p.stat + 2 * at) = make_float2(seen ? m_run : -INFINITY, l_run);
            // A part's row leaves through shared memory (every product has read what lay there) as one bulk copy: 16-byte stores of 32
            // lanes to 32 rows took 3.5 us a CTA, this 2.6.
            const int pitch = p.hd * 4 + 16;                   // (eight lanes' pieces fall into different banks)
            uint8_t* const line = smem + r * pitch;
#pragma unroll 1
            for (int c = 0; c < p.hd; c += 16) {
                uint32_t o16[16];
                if (n_blocks > 0) {                            // uniform: the load is warp-wide
                    tc_ld16(t_o + c, o16);
                    tc_ld_wait();
                }
                if (!live) continue;
                if (p.whole) {
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        w[j] = seen ? pack2(__uint_as_float(o16[2 * j]) * inv, __uint_as_float(o16[2 * j + 1]) * inv) : 0u;
                    bf16* dst = (bf16*)p.out + item * p.hd + c;
                    *(uint4*)dst = make_uint4(w[0], w[1], w[2], w[3]);
                    *(uint4*)(dst + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                } else if (seen) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) *(uint4*)(line + (c + j) * 4) = make_uint4(o16[j], o16[j + 1], o16[j + 2], o16[j + 3]);
                }
            }
            if (taken && live && seen) {
                // what was taken out of the values, for a row that sees it: its number is no longer finite
#pragma unroll 1
                for (int i = 0; i < n_blocks; ++i) {
                    if (!mixed(i)) continue;
                    const bool own = i >= seg0.n;
                    const int from = first_key_of(i) + (own ? p.prefix : 0), to = min(from + KEYS - 1, own ? pos : min(pos, p.prefix - 1));
#pragma unroll 1
                    for (int j = max(from, first); j <= to; ++j) {
                        const long long place = place_of(p, seq, j);
                        if (place < 0) continue;
                        const bf16* value = (const bf16*)p.v_pool + ((size_t)place * p.nkv + kvh) * p.hd;
#pragma unroll 2
                        for (int c = 0; c < p.hd; c += 8) {
                            const uint4 v = *(const uint4*)(value + c);
                            if (!(not_finite(v.x) || not_finite(v.y) || not_finite(v.z) || not_finite(v.w))) continue;
#pragma unroll 1
                            for (int e = c; e < c + 8; ++e) {
                                const float one = __bfloat162float(value[e]);
                                if (fabsf(one) < INFINITY) continue;
                                bf16* const result = (bf16*)p.out + item * p.hd + e;
                                if (p.whole) *result = __float2bfloat16_rn(__bfloat162float(*result) + one);
                                else ((float*)line)[e] += one;
                            }
                        }
                    }
                }
            }
            if (!p.whole && live && seen) {
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p.part + at * p.hd), "r"(smem_u32(line)),
                             "r"((uint32_t)p.hd * 4)
                             : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            }
        }
    }
    // the job's products, copies and reads are done for all roles
    blocks_before += n_blocks;
    loads_before += n_blocks > 0 ? 1 : 0;
    if (threadIdx.x == 0) {
        // the next round's pair of positions, which nobody has read since the round before this one
        s_pos[1 + 2 * (round + 1 & 1)] = 0x7fffffff;
        s_pos[2 + 2 * (round + 1 & 1)] = -1;
        s_pos[5 + 2 * THREADS + (round + 1 & 1)] = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (s_pos[0] != 0) break;                         // (the phases are no longer known)
    }
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)TMEM) : "memory");
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn() {
    static const EncodeTiled fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) ptr = nullptr;
        return (EncodeTiled)ptr;
    }();
    return fn;
}

int encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, const char* what) {
    const EncodeTiled enc = encode_fn();
    if (enc == nullptr) FR_REFUSE("attention_shared: the driver does not offer cuTensorMapEncodeTiled");
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) FR_REFUSE("attention_shared: cuTensorMapEncodeTiled failed with %d for %s", (int)r, what);
    return FR_OK;
}

int maps(const SharedArgs& p, CUtensorMap& mq, CUtensorMap& mk, CUtensorMap& mv) {
    const int G = p.nq / p.nkv;
    {
        const cuuint64_t dims[4] = {(cuuint64_t)p.hd, (cuuint64_t)G, (cuuint64_t)p.nkv, (cuuint64_t)p.rows};
        const cuuint64_t strides[3] = {(cuuint64_t)p.hd * 2, (cuuint64_t)G * p.hd * 2, (cuuint64_t)p.q_stride * 2};
        const cuuint32_t box[4] = {64, (cuuint32_t)G, 1, (cuuint32_t)(ROWS / G)};
        const int rc = encode(&mq, p.q, 4, dims, strides, box, "the queries");
        if (rc) return rc;
    }
    for (int which = 0; which < 2; ++which) {
        const cuuint64_t dims[3] = {(cuuint64_t)p.hd, (cuuint64_t)p.nkv, (cuuint64_t)p.pool_pages * PAGE};
        const cuuint64_t strides[2] = {(cuuint64_t)p.hd * 2, (cuuint64_t)p.nkv * p.hd * 2};
        const cuuint32_t box[3] = {64, 1, PAGE};
        const int rc = encode(which ? &mv : &mk, which ? p.v_pool : p.k_pool, 3, dims, strides, box, which ? "the values" : "the keys");
        if (rc) return rc;
    }
    return FR_OK;
}

int launch(const SharedArgs& p, long long jobs, cudaStream_t stream) {
    CUtensorMap mq, mk, mv;
    const int rc = maps(p, mq, mk, mv);
    if (rc) return rc;
    static std::atomic<unsigned long long> configured{0};             // a bit per device
    int device = 0;
    FR_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if (!(configured.load() & bit)) {
        FR_CUDA(cudaFuncSetAttribute(tiles_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        configured.fetch_or(bit);
    }
    const long long most = 2ll * (fr_sm_count() > 0 ? fr_sm_count() : 148);
    // (whole jobs, many of which a ragged batch does not have, are dealt out as CTAs end)
    FR_CUDA(fr_launch(tiles_kernel, dim3((unsigned)(jobs < most || p.whole ? jobs : most)), dim3(THREADS), SMEM, stream, mq, mk, mv, p));
    FR_CHECK_LAUNCH("attention_shared (tiles)");
    return FR_OK;
}

}  // namespace tcore

// ------------------------------------------------------------------ host side
struct Plan {
    int parts = 1;
    int whole = 0, prefix_splits = 0, own_splits = 0, tiles = 0, own_tiles = 0;        // tiles of all rows, of a sequence's
    long long ctas = 0;
};

// Keys a row may see in all, at most.
long long reach_of(long long max_kv_len, int window) { return window > 0 && window < max_kv_len ? window : max_kv_len; }

int clamp(long long v, long long lo, long long hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }

// The kernel of single rows: warps for two rounds of the device's, with at least 64 keys each.
Plan plan_rows(long long rows, int nq, int max_kv_len, int window) {
    Plan plan;
    const int sms = fr_sm_count();
    const long long warps = rows * nq, want = 32ll * (sms > 0 ? sms : 128), most = (reach_of(max_kv_len, window) + 63) / 64;
    plan.parts = clamp(warps > 0 ? want / warps : 1, 1, clamp(most, 1, MOST_PARTS));
    return plan;
}

// What a tile is for a call: its rows and the keys of a block, how many CTAs an SM takes, and what they cost (us; measured with one-token
// rows of 28 heads of 128, in bf16 with weights of one number): a CTA's begin and end, a block of a full tile beside others (an SM's time
// over its CTAs) and alone, and one of the rows that a sequence has.  Costs of bf16 do not go by the head size, and weights of two numbers
// add some 0.1 us to a block: what counts is which way comes out shortest, and in a sweep of forced ways over 13 bf16 shapes the choice was
// within a tenth of the best one (26.0 us for 23.8 at the worst: 8 x 20 rows behind 2,000).  float32 prompts are further off: 16 x 24 rows
// of 28 heads behind 1,000 keys are walked whole in 312 us where three shares of the prefix take 225.
struct TileKind {
    int rows = 0, keys = 0, at_once = 0;                               // rows 0: no tiles for these sizes
    double begin = 0, block = 0, alone = 0, own_block = 0, own_alone = 0;
};

TileKind kind_of(long long rows, int max_q_len, int nq, int nkv, int hd, int page, int dtype) {
    TileKind k;
    const int G = nq / nkv;
    if (dtype == FR_BF16 && hd % 16 == 0 && hd <= 128 && page == tcore::PAGE && G <= tcore::ROWS) {
        k.rows = tcore::ROWS;
        k.keys = tcore::KEYS;
        k.at_once = 2;
        k.begin = 4.0; k.block = 0.95; k.alone = 0.85; k.own_block = 0.95; k.own_alone = 1.0;
    } else if (dtype == FR_F32 && hd % 4 == 0 && hd <= 128 && G <= 64) {
        const long long heads = rows * G;                              // rows that the prefix' tiles are made of
        k.rows = heads > 32 || G > 32 ? 64 : heads > 16 || G > 16 ? 32 : 16;
        k.keys = f32::KEYS;
        k.at_once = hd <= 64 ? 3 : 2;
        const long long own = (max_q_len < k.rows / G ? max_q_len : k.rows / G) * (long long)G;
        const double steps = k.rows / 16, own_steps = own > 32 ? 4 : own > 16 ? 2 : 1, width = hd <= 32 ? 0.5 : hd <= 64 ? 1 : 2;
        k.begin = 3.0; k.alone = width * (1.6 + 0.35 * steps); k.block = width * (0.9 + 0.45 * steps);
        k.own_alone = width * (1.6 + 0.35 * own_steps); k.own_block = width * (0.9 + 0.45 * own_steps);
    }
    return k;
}

// How tiles share the work out, from an estimate of the time (us) of each way; a part of a row and head is written and read once.
Plan estimate_tiles(const TileKind& kind, long long rows, int n_seqs, int max_q_len, int max_kv_len, int prefix, int nq, int nkv, int hd, int window) {
    const double begin = kind.begin, block = kind.block, part_us = hd * 3.6e-6;
    const int sms = fr_sm_count() > 0 ? fr_sm_count() : 148;
    const int T = kind.rows / (nq / nkv);
    const long long all = (rows + T - 1) / T, own = (max_q_len + T - 1) / T;
    const double slots = (double)kind.at_once * sms, tiles = (double)(n_seqs * own < all + n_seqs ? n_seqs * own : all + n_seqs);   // that sequences' rows make
    const long long prefix_reach = window > 0 && window < prefix ? window : prefix, own_reach = reach_of(max_kv_len > prefix ? max_kv_len - prefix : 0, window);
    const long long prefix_blocks = (prefix_reach + kind.keys - 1) / kind.keys, own_blocks = (own_reach + kind.keys - 1) / kind.keys;
    Plan best;
    best.tiles = (int)all;
    best.own_tiles = (int)own;
    // whole: every CTA walks everything
    const double chain = (double)(prefix_blocks + own_blocks);
    best.whole = 1;
    best.ctas = (long long)n_seqs * nkv * own;
    double least = begin + (tiles * nkv > slots ? (double)(long long)((tiles * nkv + slots - 1) / slots) * chain * block : chain * kind.alone);
    // (one of them: as many as leave every SM one share)
    const int shares[] = {1, 2, 3, 4, 6, 8, 10, 12, 16, 20, 26, 32, 40, clamp(sms / (all * nkv), 1, 40), clamp(prefix_blocks, 1, MOST_PARTS - 8)};
    for (int os = 1; os <= 8; os *= 2) {
        if (os > 1 && os > own_blocks) break;
        for (int ps : shares) {
            if (ps > 1 && ps > prefix_blocks) continue;
            const double p_chain = (double)((prefix_blocks + ps - 1) / ps), o_chain = (double)((own_blocks + os - 1) / os);
            // (own sequences are half as long as the longest on average)
            const double total = all * nkv * (ps * begin + prefix_blocks * block) + tiles * nkv * (os * begin + 0.5 * own_blocks * kind.own_block);
            double us = total / slots;
            // (a share of the prefix beside another one on its SM, or beside own keys only)
            const double p_block = all * nkv * ps > sms ? block : kind.alone;
            if (us < begin + p_chain * p_block) us = begin + p_chain * p_block;
            if (us < begin + o_chain * kind.own_alone) us = begin + o_chain * kind.own_alone;
            us += 2.0 + rows * nq * (double)(ps + os) * part_us;
            if (us < least) {
                least = us;
                best.whole = 0;
                best.prefix_splits = ps;
                best.own_splits = os;
            }
        }
    }
    if (!best.whole) {
        best.parts = best.prefix_splits + best.own_splits;
        best.ctas = all * nkv * best.prefix_splits + (long long)n_seqs * nkv * own * best.own_splits;
    } else {
        best.prefix_splits = best.own_splits = 0;
        best.parts = 1;
    }
    return best;
}

// The same for the sizes that came before: a step's layers ask for the same way again and again.
Plan plan_tiles(const TileKind& kind, long long rows, int n_seqs, int max_q_len, int max_kv_len, int prefix, int nq, int nkv, int hd, int window) {
    const long long sizes[] = {kind.rows, kind.keys, rows, n_seqs, max_q_len, max_kv_len, prefix, nq, nkv, hd, window};
    static thread_local long long known[sizeof sizes / sizeof sizes[0]] = {};
    static thread_local Plan plan;
    if (memcmp(known, sizes, sizeof sizes) != 0) {
        plan = estimate_tiles(kind, rows, n_seqs, max_q_len, max_kv_len, prefix, nq, nkv, hd, window);
        memcpy(known, sizes, sizeof sizes);
    }
    return plan;
}

long long floats_of(const Plan& plan, long long rows, int nq, int hd) { return plan.parts > 1 ? rows * nq * plan.parts * (hd + 2) + 1 : 0; }

template <typename T>
int launch_rows(const SharedArgs& p, cudaStream_t stream) {
    const dim3 grid((unsigned)(((long long)p.rows * p.nq + 3) / 4), (unsigned)p.parts);
    if (p.hd <= 64) FR_CUDA(fr_launch(rows_kernel<T, 2>, grid, dim3(128), 0, stream, p));
    else if (p.hd <= 128) FR_CUDA(fr_launch(rows_kernel<T, 4>, grid, dim3(128), 0, stream, p));
    else FR_CUDA(fr_launch(rows_kernel<T, 8>, grid, dim3(128), 0, stream, p));
    FR_CHECK_LAUNCH("attention_shared");
    return FR_OK;
}

}  // namespace

// Working memory of a call, in floats (of whichever kernel takes it: what the queries' alignment decides is not known here).
FR_EXPORT long long attention_shared_floats(int rows, int n_seqs, int max_q_len, int max_kv_len, int prefix, int nq, int nkv, int hd,
                                            int page, int window, int dtype) {
    if (rows <= 0 || n_seqs <= 0 || nq <= 0 || nkv <= 0 || nq < nkv || hd <= 0) return 0;
    if (max_q_len > rows) max_q_len = rows;
    const long long by_rows = floats_of(plan_rows(rows, nq, max_kv_len, window), rows, nq, hd);
    const TileKind kind = kind_of(rows, max_q_len, nq, nkv, hd, page, dtype);
    if (kind.rows == 0) return by_rows;
    const long long by_tiles = floats_of(plan_tiles(kind, rows, n_seqs, max_q_len, max_kv_len, prefix, nq, nkv, hd, window), rows, nq, hd);
    return by_tiles > by_rows ? by_tiles : by_rows;
}

// seq_start, seq_qlen: per sequence its first row and its rows in this step (at most max_q_len).  max_kv_len: a bound on every row's
// position + 1, which only shares the work out.  scratch: attention_shared_floats floats.  launches: how many kernels were launched.
FR_EXPORT int attention_shared(const void* q, long long q_stride, void* out, const void* k_pool, const void* v_pool, int pool_pages, int page,
                               const int* prefix_table, int prefix, const int* block_table, int n_seqs, int table_width, const int* row_seq,
                               const int* row_pos, const int* seq_start, const int* seq_qlen, int rows, int max_q_len, int max_kv_len,
                               int nq, int nkv, int hd, int window, float scale, float* scratch, long long scratch_floats, int* status,
                               int dtype, int* launches, cudaStream_t stream) {
    *launches = 0;
    if (rows <= 0 || n_seqs <= 0) return FR_OK;
    if (dtype != FR_F32 && dtype != FR_BF16) FR_REFUSE("attention_shared: unknown dtype %d", dtype);
    if (nq < 1 || nkv < 1 || nq % nkv || hd < 1 || hd > MOST_HEAD)
        FR_REFUSE("attention_shared: %d heads on %d kv heads of %d numbers (at most %d)", nq, nkv, hd, MOST_HEAD);
    if (prefix < 0 || page < 1 || pool_pages < 1 || table_width < 0 || window < 0)
        FR_REFUSE("attention_shared: prefix %d, pages of %d, %d of them, a table %d wide, window %d", prefix, page, pool_pages, table_width, window);
    if (!(scale > 0.f) || !(scale < INFINITY)) FR_REFUSE("attention_shared: a scale of %g", (double)scale);
    if (max_q_len > rows) max_q_len = rows;                            // (a bound may be far above what there is)
    if (rows == 1) q_stride = (long long)nq * hd;                      // (of a lone row it is never used)
    SharedArgs p = {};
    p.q = q; p.out = out; p.k_pool = k_pool; p.v_pool = v_pool; p.prefix_table = prefix_table; p.block_table = block_table;
    p.row_seq = row_seq; p.row_pos = row_pos; p.q_stride = q_stride; p.rows = rows; p.n_seqs = n_seqs; p.nq = nq; p.nkv = nkv; p.hd = hd;
    p.window = window; p.prefix = prefix; p.page = page; p.pool_pages = pool_pages; p.table_width = table_width;
    p.scale_log2 = scale * 1.4426950408889634f; p.seq_start = seq_start; p.seq_qlen = seq_qlen; p.status = status;
    // Copies of 16 bytes want rows that start on 16-byte boundaries, TMA row numbers of 32 bits.
    const TileKind kind = kind_of(rows, max_q_len, nq, nkv, hd, page, dtype);
    const bool tiles = kind.rows > 0 && q_stride % (dtype == FR_BF16 ? 8 : 4) == 0 &&
                       (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0 &&
                       pool_pages < 0x7fffffff / tcore::PAGE && status != nullptr;
    const Plan plan = tiles ? plan_tiles(kind, rows, n_seqs, max_q_len, max_kv_len, prefix, nq, nkv, hd, window) : plan_rows(rows, nq, max_kv_len, window);
    if (scratch_floats < floats_of(plan, rows, nq, hd)) FR_REFUSE("attention_shared: %lld floats of working memory are too few", scratch_floats);
    if (plan.parts > 1 && (scratch == nullptr || ((uintptr_t)scratch & 15) != 0)) FR_REFUSE("attention_shared: working memory begins on a 16-byte boundary");
    p.parts = plan.parts;
    p.part = scratch;
    p.stat = scratch + ((long long)rows * nq * plan.parts * hd + 1) / 2 * 2;           // (pairs of numbers)
    if (tiles) {
        if (plan.ctas > 0x7fffffffLL) FR_REFUSE("attention_shared: %lld jobs are too many", plan.ctas);
        p.whole = plan.whole; p.prefix_splits = plan.prefix_splits; p.own_splits = plan.own_splits;
        p.jobs = (int)plan.ctas;
        p.prefix_jobs = plan.whole ? 0 : plan.tiles * nkv * plan.prefix_splits;
        p.tiles = plan.tiles; p.own_tiles = plan.own_tiles; p.tile_tokens = kind.rows / (nq / nkv);
        p.covered = plan.own_tiles * p.tile_tokens;
        p.by_tiles = FrDivide(p.tiles, p.jobs);
        p.by_kv = FrDivide(nkv, p.jobs);
        p.by_seqs = FrDivide(n_seqs, p.jobs);
        p.by_inner = FrDivide((long long)nkv * (plan.whole ? 1 : plan.own_splits), p.jobs);
        p.by_group = FrDivide(nq / nkv, kind.rows);
        p.by_prefix_splits = FrDivide(plan.whole ? 1 : plan.prefix_splits, 0x7fffffff / kind.keys + 1);
        p.by_own_splits = FrDivide(plan.whole ? 1 : plan.own_splits, 0x7fffffff / kind.keys + 1);
        const int rc = dtype == FR_BF16 ? tcore::launch(p, plan.ctas, stream)
                       : hd <= 32       ? f32::launch_rows<32>(p, kind.rows, plan.ctas, stream)
                       : hd <= 64       ? f32::launch_rows<64>(p, kind.rows, plan.ctas, stream)
                                        : f32::launch_rows<128>(p, kind.rows, plan.ctas, stream);
        if (rc != FR_OK) return rc;
    } else {
        const int rc = dtype == FR_F32 ? launch_rows<float>(p, stream) : launch_rows<bf16>(p, stream);
        if (rc != FR_OK) return rc;
    }
    *launches = 1;
    if (plan.parts > 1) {
        const dim3 grid((unsigned)((long long)rows * nq));
        p.by_heads = FrDivide(nq, (long long)rows * nq);
        p.by_pieces = FrDivide(hd % 4 == 0 ? hd / 4 : hd, 256);
        if (dtype == FR_F32 && hd % 4 == 0) FR_CUDA(fr_launch(merge_kernel<float, 4>, grid, dim3(128), 0, stream, p));
        else if (dtype == FR_F32) FR_CUDA(fr_launch(merge_kernel<float, 1>, grid, dim3(256), 0, stream, p));
        else if (hd % 4 == 0) FR_CUDA(fr_launch(merge_kernel<bf16, 4>, grid, dim3(128), 0, stream, p));
        else FR_CUDA(fr_launch(merge_kernel<bf16, 1>, grid, dim3(256), 0, stream, p));
        FR_CHECK_LAUNCH("attention_shared (merge)");
        *launches = 2;
    }
    return FR_OK;
}
