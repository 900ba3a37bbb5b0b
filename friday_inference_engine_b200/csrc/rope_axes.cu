// Rotary positions with several axes: pair i of a head turns by positions[row][a(i)] / denom[i], where a(i) is the axis (time,
// height, width) that the pair's section belongs to.  Two operations share the kernel:
//
//   rotate   `heads` heads of every row of x -> out (the same place or another)
//   append   a row is [queries | keys | values]: queries -> q_out turned, keys -> the cache's pages turned, values -> pages as they
//            are.  The place in the cache (row_seq, row_pos) and the positions that turn the heads are different numbers here, which
//            is what sets this apart from rowwise.cu's rope_kv_write: all tokens of an image share a time position.
//
// Angles.  A turn is 2^64: a pair's step per position is kept as a 64-bit fraction of a turn, 2^64 / (2 pi denom), formed in double
// precision (2 pi, its product with denom and the reciprocal are each rounded to 53 bits).  Position times step modulo 2^64 is exact for
// every 32-bit position, so what the step is off by is all that grows with the position: the angle is off by about pos / denom * 2^-52 rad,
// 2^-21 at position 2^31 with denom 1 (a float division leaves pos / denom * 2^-24, which at position 10^6 is 0.06 rad).  The upper 32
// bits go through sincospif.
#include <math.h>

#include <atomic>

#include "common.cuh"
#include "divide.cuh"
#include "tc_common.cuh"

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
    int* status;
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
    const double turns = __drcp_rn(6.283185307179586477 * (double)denom);
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

// Numbers of any size and alignment, one at a time; a block per row.
template <typename T>
__global__ void __launch_bounds__(256) rope_axes_single_kernel(const RopeArgs p) {
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

// ------------------------------------------------------------------ in pieces
// Bound by memory: every number is read and written once.  A row's work is cut into units: a piece of VEC numbers (up to 16 bytes) of a
// head's first half with the piece that it turns with (neighbours: a piece alone), then pieces that are only copied (dimensions that
// stay, values).  A block takes as many whole rows as give each of its threads up to four units, fetches all of them at once, makes the
// rows' sines and cosines (one table for all heads) while they are on the way, and ends: several blocks per SM are at different points
// of that.  The table of a row is laid out so that the lanes of one head read neighbouring 16 bytes (pairs 2 jj and 2 jj + 1 of every
// unit side by side).  Few rows are bound by the chain of launch, loads, sine and cosine: 8 rows of 36 heads of 128 into the cache 4.0 us,
// 256 rows x 32 heads of 80 3.1 us.
constexpr int AHEAD = 4, THREADS = 256, MOST_ROWS = 32;

struct Units {
    int rows, turn, stay;                             // rows of a block; where a row's units that turn end, and those that stay
    FrDivide all, half;                               // units of a row; pairs of a head
    FrDivide turn_pieces, stay_pieces, value_pieces;    // units of a head
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Piece {
    T v[VEC];
};

template <typename T, int VEC, bool NEIGHBOURS>
__global__ void __launch_bounds__(THREADS) rope_axes_kernel(const RopeArgs p, const Units un) {
    constexpr int PAIRS = NEIGHBOURS ? VEC / 2 : VEC;          // of a unit
    extern __shared__ float4 table4[];                         // per row: [PAIRS / 2][units of a head] (cos, sin, cos, sin)
    float2* table = (float2*)table4;
    __shared__ long long s_at[MOST_ROWS];                      // the row's place in the cache; -1: none, -2: the row is left alone
    typedef Piece<T, VEC> P;
    fr_pdl_wait();
    fr_pdl_launch();
    const int row0 = blockIdx.x * un.rows, rows = min(un.rows, p.rows - row0), total = rows * (int)un.all.by;
    const int turning = p.nq + p.nkv;
    struct Unit {
        int local, head, off;                                  // off: the piece's first dimension
        bool turns;
    };
    auto unit_of = [&](int idx) {
        Unit u;
        u.local = un.all.quick(idx);
        int k = idx - u.local * (int)un.all.by;
        u.turns = k < un.turn;
        if (u.turns) {
            u.head = un.turn_pieces.quick(k);
            u.off = (k - u.head * (int)un.turn_pieces.by) * VEC;
        } else if (k < un.stay) {
            k -= un.turn;
            u.head = un.stay_pieces.quick(k);
            u.off = 2 * p.half + (k - u.head * (int)un.stay_pieces.by) * VEC;
        } else {
            k -= un.stay;
            u.head = un.value_pieces.quick(k);
            u.off = (k - u.head * (int)un.value_pieces.by) * VEC;
            u.head += turning;
        }
        return u;
    };
    P a[AHEAD], b[AHEAD];
    auto fetch = [&](int base) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int idx = base + i * THREADS;
            if (idx >= total) break;
            const Unit u = unit_of(idx);
            const T* from = (const T*)p.x + (size_t)(row0 + u.local) * p.ld + (size_t)u.head * p.hd + u.off;
            a[i] = *(const P*)from;
            if (!NEIGHBOURS && u.turns) b[i] = *(const P*)(from + p.half);
        }
    };
    fetch(threadIdx.x);
    for (int idx = threadIdx.x; idx < rows * p.half; idx += THREADS) {
        const int r = un.half.quick(idx), i = idx - r * p.half, at = i / PAIRS, j = i - at * PAIRS;
        float s, c;
        sin_cos_at(turn_step(p.denom[i]), p.positions[(size_t)(row0 + r) * p.axes + axis_of(p, i)], s, c);
        table[r * p.half + (PAIRS == 1 ? at : 2 * ((j >> 1) * (int)un.turn_pieces.by + at) + (j & 1))] = make_float2(c, s);
    }
    if (threadIdx.x < rows) {
        const int row = row0 + threadIdx.x, seq = p.row_seq != nullptr ? p.row_seq[row] : 0;
        s_at[threadIdx.x] = seq < 0 ? -2 : p.nkv > 0 ? cache_row(p, seq, p.row_pos[row]) : -1;
    }
    __syncthreads();
    for (int base = threadIdx.x; base < total; base += AHEAD * THREADS) {
        if (base != (int)threadIdx.x) fetch(base);             // (rows with more units than a block's threads take at once)
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (base + i * THREADS >= total) break;
            const Unit u = unit_of(base + i * THREADS);
            const long long at = s_at[u.local];
            if (at == -2 || (u.head >= p.nq && at < 0)) continue;
            T* to;
            if (u.head < p.nq) to = (T*)p.out + (size_t)(row0 + u.local) * p.out_ld + (size_t)u.head * p.hd;
            else if (u.head < turning) to = (T*)p.k_pool + ((size_t)at * p.nkv + (u.head - p.nq)) * p.hd;
            else to = (T*)p.v_pool + ((size_t)at * p.nkv + (u.head - turning)) * p.hd;
            if (!u.turns) {
                *(P*)(to + u.off) = a[i];
                continue;
            }
            const int unit = u.off / VEC;
            float cs[2 * PAIRS];
            if (PAIRS == 1) {
                const float2 t = table[u.local * p.half + unit];
                cs[0] = t.x;
                cs[1] = t.y;
            } else {
#pragma unroll
                for (int jj = 0; jj < PAIRS / 2; ++jj) {
                    const float4 t = *(const float4*)&table[u.local * p.half + 2 * (jj * (int)un.turn_pieces.by + unit)];
                    cs[4 * jj] = t.x;
                    cs[4 * jj + 1] = t.y;
                    cs[4 * jj + 2] = t.z;
                    cs[4 * jj + 3] = t.w;
                }
            }
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                T* const x = NEIGHBOURS ? &a[i].v[2 * j] : &a[i].v[j];
                T* const y = NEIGHBOURS ? &a[i].v[2 * j + 1] : &b[i].v[j];
                float rx, ry;
                fr_rotate(fr_load(x), fr_load(y), cs[2 * j], cs[2 * j + 1], rx, ry);
                fr_store(x, rx);
                fr_store(y, ry);
            }
            *(P*)(to + u.off) = a[i];
            if (!NEIGHBOURS) *(P*)(to + u.off + p.half) = b[i];
        }
    }
}

// ------------------------------------------------------------------ many rows
// The same units, worked on in shared memory: a block goes through groups of rows, which bulk copies bring into a ring of stages and take
// from there to the queries' rows and the cache's; what is on the way never waits for what is being turned.  In a group's round its
// pieces are turned in place, the sines and cosines of the next group are made (from positions that were fetched a round before), and
// one warp sends the group off and refills the stage of the group before, a lane per row (one thread for all rows, 16 of them at most:
// 44,001 rows x 2 heads of 72, bf16, 22.4 us for 14.8; 9,000 rows of 5 heads of 32 into the cache 9.8 for 7.3).  Three blocks
// per SM with stages of up to 22 KB: 65,536 rows x 32 heads of 80, bf16, 114 us (5.9 TB/s, 0.90 of the measured copy; 133 with two blocks
// and 20 KB, 219 with the kernel above, whose blocks wait for memory, for positions and for one another in turn); 32,770 rows of 56 heads
// of 128 into the cache 164 us (352 above).
constexpr int RING_THREADS = 256, RING_BLOCKS = 3, RING_ROWS = 64;
constexpr int RING_ANGLES = 4;                                     // sines and cosines that a thread makes per group, at most
constexpr int STAGE_BYTES = 22 * 1024, RING_BYTES = 71 * 1024;     // of a group; of all stages and the tables (three blocks per SM)
// Bytes of rows: below, the kernel above.  Where the two meet differs by layout, between 0.6 and 2 MB (28 heads on 4 of 128, bf16, us, above /
// ring: 64 rows 4.08 / 3.94, 200 rows 4.5 / 4.0, 500 rows 7.3 / 5.0; 32 heads of 80: 64 rows 2.9 / 3.9, 200 rows 3.2 / 4.0, 500 rows
// 4.9 / 4.1): this bound is on the far side, so rows of 9 KB take up to 0.5 us longer than the ring would from 0.6 MB on, and no layout
// takes the ring where that is the slower way.
constexpr long long RING_FROM = 2 << 20;

__device__ __forceinline__ void bulk_in(uint32_t to, const void* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_out(void* to, uint32_t from, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(from), "r"(bytes) : "memory");
}

template <typename T, int VEC, bool NEIGHBOURS, int STAGES>
__global__ void __launch_bounds__(RING_THREADS, RING_BLOCKS) rope_axes_ring_kernel(const RopeArgs p, const Units un) {
    constexpr int PAIRS = NEIGHBOURS ? VEC / 2 : VEC;
    typedef Piece<T, VEC> P;
    extern __shared__ __align__(128) uint8_t ring[];           // [stages][rows][row bytes], then two tables of the rows' sines and cosines
    __shared__ __align__(8) uint64_t bars[STAGES];
    __shared__ unsigned long long s_step[MOST_HALF];
    __shared__ long long s_at[2][RING_ROWS];
    __shared__ unsigned char s_axis[MOST_HALF];
    const int tid = threadIdx.x, row_bytes = (p.nq + 2 * p.nkv) * p.hd * (int)sizeof(T), stage_bytes = un.rows * row_bytes;
    const uint32_t full = tc::smem_u32(bars), ring0 = tc::smem_u32(ring);
    float2* const tables = (float2*)(ring + STAGES * stage_bytes);
    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) tc::mbar_init(full + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    fr_pdl_wait();
    fr_pdl_launch();
    for (int i = tid; i < p.half; i += RING_THREADS) {
        s_step[i] = turn_step(p.denom[i]);
        s_axis[i] = (unsigned char)axis_of(p, i);
    }
    __syncthreads();
    const int groups = (p.rows + un.rows - 1) / un.rows;
    auto load = [&](int k) {                                   // the first warp's: the block's k-th group
        const long long g = (long long)blockIdx.x + (long long)k * gridDim.x;
        if (g >= groups) return;
        const int row0 = (int)g * un.rows, rows = min(un.rows, p.rows - row0), b = k % STAGES;
        if (tid == 0) tc::mbar_expect_tx(full + 8 * b, (uint32_t)(rows * row_bytes));
        __syncwarp();
        for (int r = tid; r < rows; r += 32)
            bulk_in(ring0 + (uint32_t)(b * stage_bytes + r * row_bytes), (const T*)p.x + (size_t)(row0 + r) * p.ld, (uint32_t)row_bytes, full + 8 * b);
    };
    // what a group's sines, cosines and places are made from
    int pos[RING_ANGLES], seq = -1, place = 0;
    auto fetch = [&](int k) {
        const long long g = (long long)blockIdx.x + (long long)k * gridDim.x;
        if (g >= groups) return;
        const int row0 = (int)g * un.rows, rows = min(un.rows, p.rows - row0);
#pragma unroll
        for (int i = 0; i < RING_ANGLES; ++i) {
            const int idx = tid + i * RING_THREADS;
            if (i > 0 && i * RING_THREADS >= un.rows * p.half) break;
            if (idx < rows * p.half) {
                const int r = un.half.quick(idx);
                pos[i] = p.positions[(size_t)(row0 + r) * p.axes + s_axis[idx - r * p.half]];
            }
        }
        if (tid < rows) {
            seq = p.row_seq != nullptr ? p.row_seq[row0 + tid] : 0;
            if (p.nkv > 0) place = p.row_pos[row0 + tid];
        }
    };
    auto angles = [&](int k) {
        const long long g = (long long)blockIdx.x + (long long)k * gridDim.x;
        if (g >= groups) return;
        const int row0 = (int)g * un.rows, rows = min(un.rows, p.rows - row0);
        float2* table = tables + (k & 1) * un.rows * p.half;
#pragma unroll
        for (int i = 0; i < RING_ANGLES; ++i) {
            const int idx = tid + i * RING_THREADS;
            if (i > 0 && i * RING_THREADS >= un.rows * p.half) break;
            if (idx < rows * p.half) {
                const int r = un.half.quick(idx), pair = idx - r * p.half, at = pair / PAIRS, j = pair - at * PAIRS;
                float s, c;
                sin_cos_at(s_step[pair], pos[i], s, c);
                table[r * p.half + (PAIRS == 1 ? at : 2 * ((j >> 1) * (int)un.turn_pieces.by + at) + (j & 1))] = make_float2(c, s);
            }
        }
        if (tid < rows) s_at[k & 1][tid] = seq < 0 ? -2 : p.nkv > 0 ? cache_row(p, seq, place) : -1;
    };
    if (tid < 32)
        for (int k = 0; k < STAGES - 1; ++k) load(k);
    fetch(0);
    angles(0);
    for (int k = 0;; ++k) {
        const long long g = (long long)blockIdx.x + (long long)k * gridDim.x;
        if (g >= groups) break;
        const int row0 = (int)g * un.rows, rows = min(un.rows, p.rows - row0), b = k % STAGES;
        fetch(k + 1);
        const bool here = tc::mbar_wait(full + 8 * b, (k / STAGES) & 1, p.status, 41);
        if (!__syncthreads_and(here)) break;                   // (a copy that never came: nothing more is sent)
        uint8_t* stage = ring + b * stage_bytes;
        const float2* table = tables + (k & 1) * un.rows * p.half;
        for (int idx = tid; idx < rows * un.turn; idx += RING_THREADS) {
            const int r = un.all.quick(idx), u = idx - r * un.turn, head = un.turn_pieces.quick(u), unit = u - head * (int)un.turn_pieces.by;
            T* at = (T*)(stage + r * row_bytes) + head * p.hd + unit * VEC;
            P a = *(const P*)at, b2;
            if (!NEIGHBOURS) b2 = *(const P*)(at + p.half);
#pragma unroll
            for (int jj = 0; jj < (PAIRS + 1) / 2; ++jj) {
                float4 t;
                if (PAIRS == 1) {
                    const float2 one = table[r * p.half + unit];
                    t = make_float4(one.x, one.y, 0.f, 0.f);
                } else {
                    t = *(const float4*)&table[r * p.half + 2 * (jj * (int)un.turn_pieces.by + unit)];
                }
#pragma unroll
                for (int e = 0; e < 2 && 2 * jj + e < PAIRS; ++e) {
                    const int j = 2 * jj + e;
                    T* const x = NEIGHBOURS ? &a.v[2 * j] : &a.v[j];
                    T* const y = NEIGHBOURS ? &a.v[2 * j + 1] : &b2.v[j];
                    float rx, ry;
                    fr_rotate(fr_load(x), fr_load(y), e ? t.z : t.x, e ? t.w : t.y, rx, ry);
                    fr_store(x, rx);
                    fr_store(y, ry);
                }
            }
            *(P*)at = a;
            if (!NEIGHBOURS) *(P*)(at + p.half) = b2;
        }
        angles(k + 1);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (tid < 32) {
            for (int r = tid; r < rows; r += 32) {
                const long long at = s_at[k & 1][r];
                if (at == -2) continue;
                const uint32_t from = ring0 + (uint32_t)(b * stage_bytes + r * row_bytes);
                const uint32_t q_bytes = (uint32_t)(p.nq * p.hd * (int)sizeof(T)), k_bytes = (uint32_t)(p.nkv * p.hd * (int)sizeof(T));
                if (p.nq > 0) bulk_out((T*)p.out + (size_t)(row0 + r) * p.out_ld, from, q_bytes);
                if (at < 0) continue;
                bulk_out((T*)p.k_pool + (size_t)at * p.nkv * p.hd, from + q_bytes, k_bytes);
                bulk_out((T*)p.v_pool + (size_t)at * p.nkv * p.hd, from + q_bytes + k_bytes, k_bytes);
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            // the group before has left its stage: the next group to come takes it
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            __syncwarp();
            load(k + STAGES - 1);
        }
    }
    if (tid < 32) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

int check(const RopeArgs& p, int dtype, const int* sections) {
    if (dtype != FR_F32 && dtype != FR_BF16) FR_REFUSE("rope_axes: unknown dtype %d", dtype);
    if (p.hd < 1 || p.nq < 0 || p.nkv < 0 || p.nq + p.nkv < 1) FR_REFUSE("rope_axes: %d heads, %d kv heads of %d numbers", p.nq, p.nkv, p.hd);
    if ((long long)(p.nq + 2ll * p.nkv) * p.hd > 0x3fffffffLL) FR_REFUSE("rope_axes: rows of %lld numbers", (long long)(p.nq + 2ll * p.nkv) * p.hd);
    if (p.half < 1 || p.half > MOST_HALF || 2 * p.half > p.hd)
        FR_REFUSE("rope_axes: sections of %d pairs in all do not fit heads of %d numbers (and %d pairs are the most)", p.half, p.hd, MOST_HALF);
    if (p.interleaved)
        for (int a = 1; a < p.axes; ++a)
            if (sections[a] > 0 && p.axes * (sections[a] - 1) + a >= p.half)
                FR_REFUSE("rope_axes: axis %d has %d pairs, more than its turns among %d pairs of %d axes", a, sections[a], p.half, p.axes);
    return FR_OK;
}

template <typename T, int VEC, bool NEIGHBOURS>
cudaError_t launch_pieces(const RopeArgs& p, cudaStream_t stream) {
    constexpr int PAIRS = NEIGHBOURS ? VEC / 2 : VEC;
    Units un;
    const int heads = p.nq + p.nkv, turn = p.half / PAIRS;
    const int stay = p.out == p.x && p.nkv == 0 && (p.ld == p.out_ld || p.rows == 1) ? 0 : (p.hd - 2 * p.half) / VEC;     // (in place: nothing to do)
    un.turn = heads * turn;
    un.stay = un.turn + heads * stay;
    const int all = un.stay + p.nkv * (p.hd / VEC);
    // (several rows only where all of their units are a block's)
    un.all = FrDivide(all, all > AHEAD * THREADS ? all : AHEAD * THREADS);
    un.half = FrDivide(p.half, MOST_ROWS * MOST_HALF);
    un.turn_pieces = FrDivide(turn, all);
    un.stay_pieces = FrDivide(stay > 0 ? stay : 1, all);
    un.value_pieces = FrDivide(p.hd / VEC, all);
    // as many rows as give every thread its four units, while there are more blocks than the device takes at once
    const int sms = fr_sm_count() > 0 ? fr_sm_count() : 148;
    const int fit = AHEAD * THREADS / all, spread = p.rows / (4 * sms);
    un.rows = fit < spread ? fit : spread;
    if (un.rows < 1) un.rows = 1;
    if (un.rows > MOST_ROWS) un.rows = MOST_ROWS;
    const size_t smem = (size_t)un.rows * p.half * sizeof(float2);
    return fr_launch(rope_axes_kernel<T, VEC, NEIGHBOURS>, dim3((unsigned)((p.rows + un.rows - 1) / un.rows)), dim3(THREADS), smem, stream, p, un);
}

// Many rows, each of whose ranges (queries, keys, values) is whole 16-byte pieces on 16-byte boundaries: what the ring takes.
template <typename T>
bool ring_fits(const RopeArgs& p) {
    const long long head = (long long)p.hd * (long long)sizeof(T), row_bytes = (p.nq + 2 * p.nkv) * head;
    const uintptr_t starts = (uintptr_t)p.x | (uintptr_t)p.out | (uintptr_t)p.k_pool | (uintptr_t)p.v_pool;
    const bool whole = ((p.nq * head) | (p.nkv * head) | (p.rows > 1 ? (p.ld | p.out_ld) * (long long)sizeof(T) : 0)) % 16 == 0 && starts % 16 == 0;
    return whole && row_bytes <= STAGE_BYTES && p.status != nullptr && row_bytes * p.rows >= RING_FROM;
}

template <typename T, int VEC, bool NEIGHBOURS, int STAGES>
cudaError_t launch_ring_of(const RopeArgs& p, const Units& un, int smem, cudaStream_t stream) {
    static std::atomic<unsigned long long> configured{0};                  // a bit per device
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = 1ull << (device & 63);
    if (!(configured.load() & bit)) {
        e = cudaFuncSetAttribute(rope_axes_ring_kernel<T, VEC, NEIGHBOURS, STAGES>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 RING_BYTES);
        if (e != cudaSuccess) return e;
        configured.fetch_or(bit);
    }
    const int groups = (p.rows + un.rows - 1) / un.rows, sms = fr_sm_count() > 0 ? fr_sm_count() : 148;
    return fr_launch(rope_axes_ring_kernel<T, VEC, NEIGHBOURS, STAGES>, dim3((unsigned)(groups < RING_BLOCKS * sms ? groups : RING_BLOCKS * sms)),
                     dim3(RING_THREADS), (size_t)smem, stream, p, un);
}

template <typename T, int VEC, bool NEIGHBOURS>
cudaError_t launch_ring(const RopeArgs& p, cudaStream_t stream) {
    constexpr int PAIRS = NEIGHBOURS ? VEC / 2 : VEC;
    Units un;
    const int row_bytes = (p.nq + 2 * p.nkv) * p.hd * (int)sizeof(T), turn = p.half / PAIRS;
    un.rows = STAGE_BYTES / row_bytes;
    if (un.rows > RING_ROWS) un.rows = RING_ROWS;
    // (no more rows than leave a group for every block)
    const int blocks = RING_BLOCKS * (fr_sm_count() > 0 ? fr_sm_count() : 148), share = (p.rows + blocks - 1) / blocks;
    if (un.rows > share) un.rows = share;
    if (un.rows > RING_ANGLES * RING_THREADS / p.half) un.rows = RING_ANGLES * RING_THREADS / p.half;
    // (three stages and the tables have to fit; a row's tables are at most 2 KB)
    while (un.rows > 1 && un.rows * (3 * row_bytes + 2 * p.half * (int)sizeof(float2)) > RING_BYTES) --un.rows;
    un.turn = un.stay = (p.nq + p.nkv) * turn;
    un.all = FrDivide(un.turn, (long long)un.rows * un.turn);
    un.half = FrDivide(p.half, (long long)un.rows * p.half);
    un.turn_pieces = FrDivide(turn, un.turn);
    const int stage = un.rows * row_bytes, tables = 2 * un.rows * p.half * (int)sizeof(float2);
    return 4 * stage + tables <= RING_BYTES ? launch_ring_of<T, VEC, NEIGHBOURS, 4>(p, un, 4 * stage + tables, stream)
                                            : launch_ring_of<T, VEC, NEIGHBOURS, 3>(p, un, 3 * stage + tables, stream);
}

// The widest piece (16, 8 or 4 bytes) that every head's parts, rows and starts are made of; 0: none.
template <typename T>
int piece_bytes(const RopeArgs& p) {
    if ((long long)(p.nq + 2 * p.nkv) * p.hd >= 65536) return 0;       // (FrDivide::quick: units of a row squared stay below 2^32)
    for (int bytes = 16; bytes >= 4; bytes /= 2) {
        const int vec = bytes / (int)sizeof(T);
        if (p.neighbours && vec < 2) break;
        const int pairs = p.neighbours ? vec / 2 : vec;
        const uintptr_t starts = (uintptr_t)p.x | (uintptr_t)p.out | (uintptr_t)p.k_pool | (uintptr_t)p.v_pool;
        if (p.half % pairs == 0 && p.hd % vec == 0 && (p.rows == 1 || (p.ld % vec == 0 && p.out_ld % vec == 0)) && starts % bytes == 0) return bytes;
    }
    return 0;
}

template <typename T, int VEC>
cudaError_t launch_layout(const RopeArgs& p, cudaStream_t stream) {
    const bool ring = ring_fits<T>(p);
    if constexpr (VEC >= 2)
        if (p.neighbours) return ring ? launch_ring<T, VEC, true>(p, stream) : launch_pieces<T, VEC, true>(p, stream);
    return ring ? launch_ring<T, VEC, false>(p, stream) : launch_pieces<T, VEC, false>(p, stream);
}

template <typename T>
cudaError_t launch_rows(const RopeArgs& p, cudaStream_t stream) {
    switch (piece_bytes<T>(p)) {
        case 16: return launch_layout<T, 16 / sizeof(T)>(p, stream);
        case 8: return launch_layout<T, 8 / sizeof(T)>(p, stream);
        case 4: return launch_layout<T, 4 / sizeof(T)>(p, stream);
    }
    return fr_launch(rope_axes_single_kernel<T>, dim3(p.rows), dim3(256), 0, stream, p);
}

int launch(RopeArgs& p, const int* sections, int dtype, cudaStream_t stream) {
    if (p.axes < 1 || p.axes > MOST_AXES) FR_REFUSE("rope_axes: %d axes (1 to %d)", p.axes, MOST_AXES);
    p.half = 0;
    for (int a = 0; a < p.axes; ++a) {
        if (sections[a] < 0 || sections[a] > MOST_HALF) FR_REFUSE("rope_axes: a section of %d pairs", sections[a]);
        p.half += sections[a];
        p.section_end[a] = p.interleaved ? sections[a] : p.half;
    }
    const int rc = check(p, dtype, sections);
    if (rc || p.rows <= 0) return rc;
    if (dtype == FR_F32) FR_CUDA(launch_rows<float>(p, stream));
    else FR_CUDA(launch_rows<__nv_bfloat16>(p, stream));
    FR_CHECK_LAUNCH("rope_axes");
    return FR_OK;
}

}  // namespace

// x: rows of ld elements, head h at h * hd; out likewise (out == x with the same row length: in place).  positions [rows][axes];
// denom [sum of sections]; sections: host, [axes].
FR_EXPORT int rope_axes_rotate(const void* x, long long ld, void* out, long long out_ld, int rows, int heads, int hd, const int* positions,
                               int axes, const float* denom, const int* sections, int interleaved, int neighbours, int* status, int dtype,
                               cudaStream_t stream) {
    RopeArgs p = {};
    p.x = x; p.ld = ld; p.out = out; p.out_ld = out_ld; p.rows = rows; p.nq = heads; p.hd = hd; p.positions = positions; p.axes = axes;
    p.denom = denom; p.interleaved = interleaved != 0; p.neighbours = neighbours != 0; p.status = status;
    return launch(p, sections, dtype, stream);
}

// qkv: rows of ld elements, [nq | nkv | nkv] heads of hd.  Rows whose row_seq is negative are left alone (their queries too); a row
// whose place the table does not name (a position beyond it, a negative page, a page beyond the pool) only gets its queries.
FR_EXPORT int rope_axes_append(const void* qkv, long long ld, void* q_out, long long q_ld, int rows, int nq, int nkv, int hd,
                               const int* row_seq, const int* row_pos, const int* positions, int axes, const float* denom,
                               const int* sections, int interleaved, int neighbours, void* k_pool, void* v_pool, int pool_pages, int page,
                               const int* block_table, int n_seqs, int table_width, int* status, int dtype, cudaStream_t stream) {
    RopeArgs p = {};
    if (nkv < 1 || page < 1 || table_width < 1 || n_seqs < 1 || pool_pages < 1)
        FR_REFUSE("rope_axes: a cache of %d pages of %d rows, %d kv heads, a table of %d x %d", pool_pages, page, nkv, n_seqs, table_width);
    p.x = qkv; p.ld = ld; p.out = q_out; p.out_ld = q_ld; p.rows = rows; p.nq = nq; p.nkv = nkv; p.hd = hd; p.row_seq = row_seq;
    p.row_pos = row_pos; p.positions = positions; p.axes = axes; p.denom = denom; p.interleaved = interleaved != 0;
    p.neighbours = neighbours != 0; p.k_pool = k_pool; p.v_pool = v_pool; p.pool_pages = pool_pages; p.page = page;
    p.block_table = block_table; p.n_seqs = n_seqs; p.table_width = table_width; p.status = status;
    return launch(p, sections, dtype, stream);
}
