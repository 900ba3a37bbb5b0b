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

#include <stdlib.h>

#include <atomic>

#include "common.cuh"
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
    int prefix_ctas, prefix_splits, own_splits;           // prefix_splits 0: parts are not of one range or the other
    int covered;              // rows of a sequence that the grid's own tiles reach
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
    // own parts are there for rows that the sequence's range names
    int parts = p.parts;
    if (p.prefix_splits > 0) {
        const int t = row - p.seq_start[seq];
        if (t < 0 || t >= min(p.seq_qlen[seq], p.covered)) parts = p.prefix_splits;
    }
    // lane s has the statistics of parts s and s + 32
    const float* stat = p.stat + 2 * (size_t)item * p.parts;
    float m[2], l[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool there = lane + 32 * i < parts;
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
    for (int s = 0; s < parts; ++s) {
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

// ------------------------------------------------------------------ bf16 on the tensor cores
// Both products are tcgen05.mma with scores, weights and results in tensor memory.  A tile is 128 rows of one kv head; row r of it
// stands for (token row r / G, group head r % G), G = heads / kv heads.  For the prefix a tile's token rows are any consecutive rows
// of the step, whatever sequences they belong to: that is what reads the prefix once for all.  For own keys they are rows of one
// sequence.  A CTA has TILES tiles that share the blocks of keys it walks, and one of three jobs:
//
//   prefix   consecutive rows of the step, a share of the prefix' blocks            -> a part
//   own      rows of one sequence, a share of its own blocks                        -> a part
//   whole    rows of one sequence, all of the prefix' blocks and then its own       -> the result (many rows per sequence)
//
//   warp 0      TMA: the queries (a 4-d box [64 dims][G heads][1][T rows] per 64-dim slice lands as rows t * G + g, 128-byte
//               swizzle), then K of the block after and V of this one; a page that a table leaves out, or that lies behind the last
//               key in sight, is loaded from beyond the pool's last row, which fills zeros
//   warp 1      tensor memory; one lane issues S = Q K^T and O += P V
//   four warps  per tile, one thread per row: maximum, exponentials, running maximum and sum; P goes back into tensor memory as bf16
//               over its scores.  The reference maximum only moves when the true one has grown by more than 8 (in log2 units; weights
//               stay below 2^8); O is rescaled then.
//
// TILES 1: blocks of 64 keys, two stages of scores, half the tensor memory, two CTAs per SM.  TILES 2: blocks of 128 keys, one stage
// of scores per tile, the tiles take turns on the tensor core.  P is rounded to bf16 for the second product (its sum is not); scores,
// sums and results are 32-bit.  Values of positions that no row of the CTA sees may be anything: their rows are zeroed in shared
// memory before the product.  (A position that one row sees and another does not must hold finite values: zero times infinity.)
// Every wait on an mbarrier is bounded; a wait that gives up leaves a code in `status` and all roles leave their loops.
namespace tcore {

using namespace tc;

constexpr int ROWS = 128, PAGE = 64;
constexpr int SLICE = ROWS * 128;         // bytes of 128 rows of 64 numbers

template <int TILES>
struct Shape {
    static constexpr int KEYS = TILES == 2 ? 128 : 64, PAGES = KEYS / PAGE, THREADS = 64 + 128 * TILES;
    static constexpr int KSLICE = KEYS * 128, STAGE = 2 * KSLICE;              // a block's keys (or values): two slices of 64 dims
    static constexpr int TMEM = TILES == 2 ? 512 : 256;
    static constexpr int SMEM = 2 * TILES * SLICE + 4 * STAGE + 1024 + 256;
    // columns: TILES 2: tile x has S at 256 x (P over its first half) and O behind it; TILES 1: S of even blocks, S of odd blocks, O
};

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
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, "
        "%25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
          "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
          "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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
// D[tmem] (+)= A[tmem] * B[smem]: lane = row, two bf16 per column of A
__device__ __forceinline__ void mma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// a row's position, no further than the tables have room; -1: it sees nothing
__device__ __forceinline__ int position_of(const SharedArgs& p, int row) {
    const long long room = (long long)p.prefix + (long long)p.table_width * PAGE;
    return max(-1, (int)min((long long)p.row_pos[row], room - 1));
}

// Keys [lo, hi] of a range of pages that the CTA's rows see between them (none: hi < lo), block `first` its first one here, n blocks.
struct Range {
    int lo, hi, first, n;
};

template <int TILES>
__global__ void __launch_bounds__(Shape<TILES>::THREADS, TILES == 2 ? 1 : 2)
tiles_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
             const SharedArgs p) {
    typedef Shape<TILES> S;
    constexpr int KEYS = S::KEYS, KSLICE = S::KSLICE, STAGE = S::STAGE;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* s_q = smem;                              // [tiles][2 slices][128 rows][128 B]
    uint8_t* s_k = s_q + 2 * TILES * SLICE;           // [2 stages][2 slices][KEYS][128 B]
    uint8_t* s_v = s_k + 2 * STAGE;
    uint64_t* bars = (uint64_t*)(s_v + 2 * STAGE);
    // bars: q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], pv_done[2]
    uint32_t* tmem_slot = (uint32_t*)(bars + 15);
    int* s_pos = (int*)(tmem_slot + 1);               // [2 tiles][least, greatest position of a live row]

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
            s_pos[2 * b] = 0x7fffffff;
            s_pos[2 * b + 1] = -1;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)S::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    fr_pdl_wait();
    if (threadIdx.x == 0) fr_pdl_launch();

    // The CTA's job.  Tiles of one kv head and share of the prefix are neighbours in the grid: they read the same pages at about the
    // same time.  CTAs start in the order of their index: the prefix' shares (the most work) first, a whole job's late rows first.
    const int G = p.nq / p.nkv, T = ROWS / G;         // token rows of a tile
    const bool prefix_job = !p.whole && (int)blockIdx.x < p.prefix_ctas;
    int kvh, seq = 0, group, part, share, shares;     // group: which TILES tiles of the rows
    int begin = 0, count = p.rows;                    // the rows that the tiles are taken from
    if (prefix_job) {
        const int per = p.prefix_ctas / (p.nkv * p.prefix_splits);
        group = blockIdx.x % per;
        kvh = blockIdx.x / per % p.nkv;
        share = blockIdx.x / (per * p.nkv);
        shares = p.prefix_splits;
        part = share;
    } else {
        const int x = blockIdx.x - (p.whole ? 0 : p.prefix_ctas), splits = p.whole ? 1 : p.own_splits;
        const int per = (gridDim.x - (p.whole ? 0 : p.prefix_ctas)) / (p.n_seqs * p.nkv * splits);
        seq = x % p.n_seqs;
        kvh = x / p.n_seqs % p.nkv;
        share = x / (p.n_seqs * p.nkv) % splits;
        group = per - 1 - x / (p.n_seqs * p.nkv * splits);
        shares = splits;
        part = p.prefix_splits + share;
        begin = p.seq_start[seq];
        count = p.seq_qlen[seq];
        if (begin < 0 || begin > p.rows) count = 0;
        else count = min(count, p.rows - begin);
    }
    int row0[TILES], n_tok[TILES];
    bool active[TILES];
#pragma unroll
    for (int x = 0; x < TILES; ++x) {
        const int t0 = (group * TILES + x) * T;
        row0[x] = begin + t0;
        n_tok[x] = max(0, min(T, count - t0));
        for (int t = threadIdx.x; t < n_tok[x]; t += S::THREADS) {
            const int of = p.row_seq[row0[x] + t];
            if (of >= 0 && of < p.n_seqs) {
                const int pos = position_of(p, row0[x] + t);
                atomicMin(&s_pos[2 * x], pos);
                atomicMax(&s_pos[2 * x + 1], pos);
            }
        }
    }
    __syncthreads();
    int least = 0x7fffffff, most = -1;
#pragma unroll
    for (int x = 0; x < TILES; ++x) {
        active[x] = s_pos[2 * x + 1] >= 0;
        least = min(least, s_pos[2 * x]);
        most = max(most, s_pos[2 * x + 1]);
    }
    Range seg[2];                                     // of the prefix, of own keys (numbered from the prefix' end)
    {
        const int lo = most < 0 ? 0 : fr_first_key(least, p.window, 0);
        seg[0] = Range{lo, (p.whole || prefix_job) ? min(most, p.prefix - 1) : -1, 0, 0};
        seg[1] = Range{max(0, lo - p.prefix), prefix_job ? -1 : most - p.prefix, 0, 0};
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (seg[g].hi < seg[g].lo) continue;
            const int first = seg[g].lo / KEYS, n = seg[g].hi / KEYS - first + 1;
            const int from = (int)((long long)n * share / shares), to = (int)((long long)n * (share + 1) / shares);
            seg[g].first = first + from;
            seg[g].n = to - from;
        }
    }
    const int n_blocks = seg[0].n + seg[1].n;
    const int slices = (p.hd + 63) / 64;
    auto first_key_of = [&](int i) { return (i < seg[0].n ? seg[0].first + i : seg[1].first + i - seg[0].n) * KEYS; };

    // Block i uses stage i & 1 of K and V, in their (i >> 1)-th use.
    if (warp == 0) {
        if (n_blocks > 0 && elect_one()) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
            int there = 0;
            for (int x = 0; x < TILES; ++x) there += active[x] ? 1 : 0;
            mbar_expect_tx(q_full, (uint32_t)(there * slices * 64 * G * T * 2));
            for (int x = 0; x < TILES; ++x)
                if (active[x])
                    for (int s = 0; s < slices; ++s)
                        load_4d(smem_u32(s_q + (2 * x + s) * SLICE), &map_q, s * 64, 0, kvh, row0[x], q_full);
            auto load = [&](int i, const CUtensorMap* map, uint8_t* ring, uint32_t full, uint32_t empty) {
                const int b = i & 1, par = (i >> 1) & 1;
                if (!mbar_wait(empty + 8 * b, par ^ 1, p.status, 1)) return false;
                mbar_expect_tx(full + 8 * b, (uint32_t)(S::PAGES * slices * PAGE * 128));
                const bool own = i >= seg[0].n;
                const int j0 = first_key_of(i), hi = own ? seg[1].hi : seg[0].hi;
                const int* table = own ? p.block_table + (size_t)seq * p.table_width : p.prefix_table;
#pragma unroll
                for (int pg = 0; pg < S::PAGES; ++pg) {
                    const int j = j0 + pg * PAGE;
                    int page = j <= hi ? table[j / PAGE] : -1;
                    if (page < 0 || page >= p.pool_pages) page = p.pool_pages;          // beyond the pool: zeros
                    for (int s = 0; s < slices; ++s)
                        load_3d(smem_u32(ring) + (uint32_t)(b * STAGE + s * KSLICE + pg * PAGE * 128), map, s * 64, kvh, page * PAGE, full + 8 * b);
                }
                return true;
            };
            bool ok = load(0, &map_k, s_k, k_full, k_empty);
            for (int i = 0; i < n_blocks && ok; ++i) {
                if (i + 1 < n_blocks) ok = load(i + 1, &map_k, s_k, k_full, k_empty);
                if (ok) ok = load(i, &map_v, s_v, v_full, v_empty);
            }
        }
    } else if (warp == 1) {
        if (n_blocks > 0 && elect_one()) {
            const uint32_t idesc_qk = instr_desc(ROWS, KEYS);
            const uint32_t idesc_pv = instr_desc(ROWS, p.hd) | (1u << 16);              // B is MN-major
            const int k_steps = p.hd / 16;
            bool ok = mbar_wait(q_full, 0, p.status, 2);
            // (descriptors are made once and stepped: a lone thread issues all of this)
            const uint64_t dq0 = smem_desc(smem_u32(s_q)), dk0 = smem_desc(smem_u32(s_k)), dv0 = desc_mn(smem_u32(s_v), KSLICE, 1024);
            auto scores = [&](int x, int i) {
                const int b = i & 1, par = (i >> 1) & 1;
                if (!mbar_wait(k_full + 8 * b, par, p.status, 3)) return false;
                tc_fence_after();
                uint64_t da = dq0 + (uint64_t)(x * (2 * SLICE >> 4)), db = dk0 + (uint64_t)(b * (STAGE >> 4));
                const uint32_t d = tmem + (TILES == 2 ? 256 * x : KEYS * b);
                for (int ks = 0; ks < k_steps; ++ks) {
                    tc_mma(d, da, db, idesc_qk, ks > 0 ? 1u : 0u);
                    // 32 bytes on in the 128-byte row; after four of them the next slice of 64 dims
                    da += (ks & 3) == 3 ? (uint64_t)((SLICE >> 4) - 6) : 2ull;
                    db += (ks & 3) == 3 ? (uint64_t)((KSLICE >> 4) - 6) : 2ull;
                }
                tc_commit(s_full + 8 * (TILES == 2 ? x : b));
                return true;
            };
            auto second = [&](int x, int i) {
                const int b = i & 1, par = (i >> 1) & 1;
                if (!mbar_wait(v_full + 8 * b, par, p.status, 4)) return false;
                // P of block i: the tile's i-th (TILES 2), or the stage's (i >> 1)-th
                if (!mbar_wait(p_full + 8 * (TILES == 2 ? x : b), TILES == 2 ? i & 1 : par, p.status, 5)) return false;
                tc_fence_after();
                const int hi = i < seg[0].n ? seg[0].hi : seg[1].hi;
                const int steps = (min(KEYS, hi - first_key_of(i) + 1) + 15) / 16;
                uint64_t db = dv0 + (uint64_t)(b * (STAGE >> 4));
                uint32_t pa = tmem + (TILES == 2 ? 256 * x : KEYS * b), keep = i > 0 ? 1u : 0u;
                const uint32_t d = tmem + (TILES == 2 ? 256 * x + 128 : 128);
                for (int ks = 0; ks < steps; ++ks) {
                    mma_ta(d, pa, db, idesc_pv, keep);
                    keep = 1u;
                    pa += 8;                                   // 16 keys of P: 8 columns
                    db += (uint64_t)(16 * 128 >> 4);           // 16 keys of V
                }
                return true;
            };
            if (TILES == 2) {
                for (int x = 0; x < TILES && ok; ++x)
                    if (active[x]) ok = scores(x, 0);
                if (ok) tc_commit(k_empty);
                for (int i = 0; i < n_blocks && ok; ++i) {
                    for (int x = 0; x < TILES && ok; ++x) {
                        if (!active[x]) continue;
                        ok = second(x, i);
                        if (ok && i + 1 < n_blocks) ok = scores(x, i + 1);
                    }
                    if (!ok) break;
                    tc_commit(v_empty + 8 * (i & 1));
                    if (i + 1 < n_blocks) tc_commit(k_empty + 8 * ((i + 1) & 1));
                }
                if (ok) tc_commit(pv_done);
            } else {
                // the scores run two blocks ahead of the second product
                for (int i = 0; i < 2 && i < n_blocks && ok; ++i) {
                    ok = scores(0, i);
                    if (ok) tc_commit(k_empty + 8 * (i & 1));
                }
                for (int i = 0; i < n_blocks && ok; ++i) {
                    ok = second(0, i);
                    if (!ok) break;
                    tc_commit(pv_done + 8 * (i & 1));
                    tc_commit(v_empty + 8 * (i & 1));
                    if (i + 2 < n_blocks) {
                        ok = scores(0, i + 2);
                        if (ok) tc_commit(k_empty + 8 * (i & 1));
                    }
                }
            }
        }
    } else {
        const int x = TILES == 2 ? (warp - 2) >> 2 : 0;
        const int quarter = warp & 3;                          // the tensor-memory lanes that this warp may touch: 32 * quarter ..
        const int r = quarter * 32 + lane, t = r / G, g = r - t * G;
        const int row = row0[x] + t;
        int pos = -1;
        bool live = r < T * G && t < n_tok[x];
        if (live) {
            const int of = p.row_seq[row];
            live = of >= 0 && of < p.n_seqs;
            if (live) pos = position_of(p, row);
        }
        const int first = fr_first_key(pos, p.window, 0);
        const bool any = __any_sync(0xffffffffu, live && pos >= 0);       // a warp without rows only keeps the barriers going
        const int tile_least = s_pos[2 * x], tile_first_max = fr_first_key(s_pos[2 * x + 1], p.window, 0);
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        const uint32_t t_o = tmem + lane_addr + (TILES == 2 ? 256 * x + 128 : 128);
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        const int mine = active[x] ? n_blocks : 0;
        for (int i = 0; i < mine; ++i) {
            const int b = i & 1, par = (i >> 1) & 1;
            const bool own = i >= seg[0].n;
            const int j0 = first_key_of(i), base = own ? p.prefix : 0;
            if (!(ok = mbar_wait(s_full + 8 * (TILES == 2 ? x : b), TILES == 2 ? i & 1 : par, p.status, 6))) break;
            tc_fence_after();
            const uint32_t t_s = tmem + lane_addr + (TILES == 2 ? 256 * x : KEYS * b);
            if (any) {
                uint32_t raw[KEYS];
#pragma unroll
                for (int c = 0; c < KEYS / 32; ++c) ld32(t_s + 32 * c, &raw[32 * c]);
                tc_ld_wait();
                // columns hi < j or j < lo are masked; the choice is the tile's
                const int hi = own ? pos - p.prefix - j0 : min(pos, p.prefix - 1) - j0, lo = first - base - j0;
                const bool need_mask = j0 + KEYS - 1 > (own ? tile_least - p.prefix : min(tile_least, p.prefix - 1)) || j0 < tile_first_max - base;
                if (need_mask) {
#pragma unroll
                    for (int j = 0; j < KEYS; ++j)
                        if (j > hi || j < lo) raw[j] = 0xff800000u;      // -inf
                }
                // (the maximum in four strands; the positive scale is applied to the result)
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < KEYS; ++j) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(raw[j]));
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
                const bool grow = mx > m_run + 8.f;
                if (__any_sync(0xffffffffu, grow)) {
                    const float alpha = grow ? exp2f(m_run - mx) : 1.f;      // 0 for a row that had seen no key
                    if (grow) {
                        m_run = mx;
                        l_run *= alpha;
                    }
                    if (i > 0) {
                        // Every product into O so far must be done.  TILES 2: this block's scores were issued behind them.  TILES 1:
                        // those of block i - 2 likewise, so the wait for the other stage's phase is unambiguous.
                        if (TILES == 1) {
                            if (!(ok = mbar_wait(pv_done + 8 * (b ^ 1), ((i - 1) >> 1) & 1, p.status, 8))) break;
                            tc_fence_after();
                        }
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
                float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int h = 0; h < KEYS / 64; ++h) {
                    uint32_t packed[32];
#pragma unroll
                    for (int j = 0; j < 64; j += 2) {
                        const float e0 = exp2_fast(fmaf(__uint_as_float(raw[64 * h + j]), p.scale_log2, neg_m));
                        const float e1 = exp2_fast(fmaf(__uint_as_float(raw[64 * h + j + 1]), p.scale_log2, neg_m));
                        sum4[j & 2] += e0;
                        sum4[(j & 2) + 1] += e1;
                        packed[j >> 1] = pack2(e0, e1);
                    }
                    st32(t_s + 32 * h, packed);
                }
                st_wait();
                l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
            }
            const Range& here = seg[own ? 1 : 0];
            if (j0 < here.lo || j0 + KEYS - 1 > here.hi) {
                // positions that no row of the CTA sees: their values may be anything (both tiles do this, each before it hands over
                // its P of this block)
                if (!(ok = mbar_wait(v_full + 8 * b, par, p.status, 7))) break;
                if (r < KEYS && (j0 + r < here.lo || j0 + r > here.hi)) {
                    for (int s = 0; s < slices; ++s) {
                        uint4* line = (uint4*)(s_v + b * STAGE + s * KSLICE + r * 128);
#pragma unroll
                        for (int q = 0; q < 8; ++q) line[q] = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            }
            tc_fence_before();
            mbar_arrive(p_full + 8 * (TILES == 2 ? x : b));
        }
        if (ok && mine > 0) {
            ok = TILES == 2 ? mbar_wait(pv_done, 0, p.status, 8) : mbar_wait(pv_done + 8 * ((mine - 1) & 1), ((mine - 1) >> 1) & 1, p.status, 8);
            tc_fence_after();
        }
        if (ok) {
            const size_t item = (size_t)row * p.nq + (size_t)kvh * G + g;
            const bool seen = l_run != 0.f;                    // (a NaN is seen)
            if (p.whole) {
                const float inv = l_run > 0.f ? 1.f / l_run : l_run;
                bf16* dst = (bf16*)p.out + item * p.hd;
#pragma unroll 1
                for (int c = 0; c < p.hd; c += 16) {
                    uint32_t o16[16];
                    if (mine > 0) {                            // uniform: the load is warp-wide
                        tc_ld16(t_o + c, o16);
                        tc_ld_wait();
                    }
                    if (live) {
                        uint32_t w[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            w[j] = seen ? pack2(__uint_as_float(o16[2 * j]) * inv, __uint_as_float(o16[2 * j + 1]) * inv) : 0u;
                        *(uint4*)(dst + c) = make_uint4(w[0], w[1], w[2], w[3]);
                        *(uint4*)(dst + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
            } else {
                const size_t at = item * p.parts + part;
                if (live) *(float2*)(p.stat + 2 * at) = make_float2(seen ? m_run : -INFINITY, l_run);
                float* dst = p.part + at * p.hd;
                if (mine > 0 && any) {
#pragma unroll 1
                    for (int c = 0; c < p.hd; c += 16) {
                        uint32_t o16[16];
                        tc_ld16(t_o + c, o16);
                        tc_ld_wait();
                        if (live && seen) {
#pragma unroll
                            for (int j = 0; j < 16; j += 4)
                                *(float4*)(dst + c + j) = make_float4(__uint_as_float(o16[j]), __uint_as_float(o16[j + 1]), __uint_as_float(o16[j + 2]),
                                                                      __uint_as_float(o16[j + 3]));
                        }
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)S::TMEM) : "memory");
    }
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
        // (the stride between rows of a lone row is never used, but has to be one that a map takes)
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

template <int TILES>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const SharedArgs& p, long long ctas, cudaStream_t stream) {
    static std::atomic<unsigned long long> configured{0};             // a bit per device
    int device = 0;
    FR_CUDA(cudaGetDevice(&device));
    const unsigned long long bit = 1ull << (device & 63);
    if (!(configured.load() & bit)) {
        FR_CUDA(cudaFuncSetAttribute(tiles_kernel<TILES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<TILES>::SMEM));
        configured.fetch_or(bit);
    }
    FR_CUDA(fr_launch(tiles_kernel<TILES>, dim3((unsigned)ctas), dim3(Shape<TILES>::THREADS), Shape<TILES>::SMEM, stream, mq, mk, mv, p));
    FR_CHECK_LAUNCH("attention_shared (tiles)");
    return FR_OK;
}

}  // namespace tcore

// ------------------------------------------------------------------ host side
struct Plan {
    int parts = 1;
    int tiles = 0;                                    // 0: the kernel of single rows; 1, 2: tiles per CTA of the tensor-core kernel
    int whole = 0, prefix_splits = 0, own_splits = 0, groups = 0, own_groups = 0;      // groups of `tiles` tiles: of all rows, of a sequence's
    long long ctas = 0;
};

// Keys a row may see in all, at most.
long long reach_of(int max_kv_len, int window) { return window > 0 && window < max_kv_len ? window : max_kv_len; }

int clamp(long long v, long long lo, long long hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }

// The kernel of single rows: warps for two rounds of the device's, with at least 64 keys each.
Plan plan_rows(long long rows, int nq, int max_kv_len, int window) {
    Plan plan;
    const int sms = fr_sm_count();
    const long long warps = rows * nq, want = 32ll * (sms > 0 ? sms : 128), most = (reach_of(max_kv_len, window) + 63) / 64;
    plan.parts = clamp(warps > 0 ? want / warps : 1, 1, clamp(most, 1, MOST_PARTS));
    return plan;
}

bool tiles_fit(int nq, int nkv, int hd, int page, int dtype) {
    return dtype == FR_BF16 && hd % 16 == 0 && hd <= 128 && page == tcore::PAGE && nq / nkv <= tcore::ROWS;
}

Plan plan_tiles(long long rows, int n_seqs, int max_q_len, int max_kv_len, int prefix, int nq, int nkv, int window) {
    Plan plan;
    const int sms = fr_sm_count() > 0 ? fr_sm_count() : 148;
    const int T = tcore::ROWS / (nq / nkv);
    const long long all = (rows + T - 1) / T, own = (max_q_len + T - 1) / T;
    int tiles = all > 1 ? 2 : 1, whole = 0, ps = -1, os = -1;
    if (const char* e = getenv("FRIDAY_SHARED_PLAN")) sscanf(e, "%d,%d,%d,%d", &tiles, &whole, &ps, &os);
    plan.tiles = tiles;
    plan.groups = (int)((all + tiles - 1) / tiles);
    plan.own_groups = (int)((own + tiles - 1) / tiles);
    const int keys = tiles == 2 ? 128 : 64;
    const long long slots = (long long)sms * (tiles == 2 ? 1 : 2);
    const long long prefix_reach = window > 0 && window < prefix ? window : prefix, own_reach = reach_of(max_kv_len - prefix, window);
    const long long prefix_blocks = (prefix_reach + keys - 1) / keys, own_blocks = (own_reach + keys - 1) / keys;
    if (whole) {
        plan.whole = 1;
        plan.ctas = (long long)n_seqs * nkv * plan.own_groups;
        return plan;
    }
    const long long n_prefix = (long long)plan.groups * nkv;
    plan.prefix_splits = ps > 0 ? ps : clamp(slots / n_prefix, 1, clamp(prefix_blocks, 1, 40));
    const long long each = (prefix_blocks + plan.prefix_splits - 1) / plan.prefix_splits;
    plan.own_splits = os > 0 ? os : clamp(own_blocks / (each > 4 ? each : 4), 1, 16);
    plan.parts = plan.prefix_splits + plan.own_splits;
    plan.ctas = n_prefix * plan.prefix_splits + (long long)n_seqs * nkv * plan.own_groups * plan.own_splits;
    return plan;
}

long long floats_of(const Plan& plan, long long rows, int nq, int hd) { return plan.parts > 1 ? rows * nq * plan.parts * (hd + 2) : 0; }

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
    const long long by_rows = floats_of(plan_rows(rows, nq, max_kv_len, window), rows, nq, hd);
    if (!tiles_fit(nq, nkv, hd, page, dtype)) return by_rows;
    const long long by_tiles = floats_of(plan_tiles(rows, n_seqs, max_q_len, max_kv_len, prefix, nq, nkv, window), rows, nq, hd);
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
    SharedArgs p = {};
    p.q = q; p.out = out; p.k_pool = k_pool; p.v_pool = v_pool; p.prefix_table = prefix_table; p.block_table = block_table;
    p.row_seq = row_seq; p.row_pos = row_pos; p.q_stride = q_stride; p.rows = rows; p.n_seqs = n_seqs; p.nq = nq; p.nkv = nkv; p.hd = hd;
    p.window = window; p.prefix = prefix; p.page = page; p.pool_pages = pool_pages; p.table_width = table_width;
    p.scale_log2 = scale * 1.4426950408889634f; p.seq_start = seq_start; p.seq_qlen = seq_qlen; p.status = status;
    // TMA wants rows that start on 16-byte boundaries, and row numbers of 32 bits
    const bool tiles = tiles_fit(nq, nkv, hd, page, dtype) && q_stride % 8 == 0 &&
                       (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15) == 0 &&
                       pool_pages < 0x7fffffff / tcore::PAGE && status != nullptr;
    const Plan plan = tiles ? plan_tiles(rows, n_seqs, max_q_len, max_kv_len, prefix, nq, nkv, window) : plan_rows(rows, nq, max_kv_len, window);
    if (scratch_floats < floats_of(plan, rows, nq, hd)) FR_REFUSE("attention_shared: %lld floats of working memory are too few", scratch_floats);
    p.parts = plan.parts;
    p.part = scratch;
    p.stat = scratch + (long long)rows * nq * plan.parts * hd;
    if (tiles) {
        const int T = tcore::ROWS / (nq / nkv);
        p.whole = plan.whole; p.prefix_splits = plan.prefix_splits; p.own_splits = plan.own_splits;
        p.prefix_ctas = plan.whole ? 0 : plan.groups * nkv * plan.prefix_splits;
        p.covered = plan.own_groups * plan.tiles * T;
        CUtensorMap mq, mk, mv;
        int rc = tcore::maps(p, mq, mk, mv);
        if (rc == FR_OK) rc = plan.tiles == 2 ? tcore::launch<2>(mq, mk, mv, p, plan.ctas, stream) : tcore::launch<1>(mq, mk, mv, p, plan.ctas, stream);
        if (rc != FR_OK) return rc;
    } else {
        const int rc = dtype == FR_F32 ? launch_rows<float>(p, stream) : launch_rows<bf16>(p, stream);
        if (rc != FR_OK) return rc;
    }
    *launches = 1;
    if (plan.parts > 1) {
        const dim3 grid((unsigned)(((long long)rows * nq + 3) / 4));
        if (dtype == FR_F32) FR_CUDA(fr_launch(merge_kernel<float>, grid, dim3(128), 0, stream, p));
        else FR_CUDA(fr_launch(merge_kernel<bf16>, grid, dim3(128), 0, stream, p));
        FR_CHECK_LAUNCH("attention_shared (merge)");
        *launches = 2;
    }
    return FR_OK;
}
