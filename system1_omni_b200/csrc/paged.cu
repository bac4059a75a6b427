// Full attention of the tokens after a prefill, over a cache kept in pages: norm, rotary and gate split
// of new rows with their keys and values put into the cache, and the attention of new rows over it.
//
// A cache is two pools [n_pages, page_tokens, Hk, Dh] (keys after norm and rotary, values as
// projected) and a table [sequences, table_pages] of page numbers: token p of a sequence is row
// p % page_tokens of page table[p / page_tokens]. Several sequences may name the same page.
//
// Float32 from the inputs to one rounding at the end (the prefill's operators round in between where
// the model stores a tensor, and their attention the probabilities to bf16, so bf16 results may differ from theirs
// by a step). The probabilities go into the product with the values as two bf16 terms, off by
// 2^-15 of their float32 values at most.
#include <math.h>

#include <algorithm>

#include "common.cuh"
#include "cs1_ops.h"
#include "s1_executor.h"
#include "status.h"
#include "tc5.cuh"
#include "tmap.h"

namespace s1 {
namespace {

using namespace tc5;

// Codes left in the attention step operators' device error word.
enum { PAGED_WAIT = 30, PAGED_BAD_ROW = 31, PAGED_BAD_PAGE = 32, PAGED_BAD_ANGLE = 33, PAGED_CLASH = 34 };

struct PageTable {
    const int* pages;  // [sequences, width]
    int width, sequences, n_pages, page_tokens;
};

// ---- q/k RMSNorm + rotary + gate split + cache append ----
struct PrepArgs {
    const bf16 *qg, *kr, *vr, *qw, *kw, *cos, *sin;
    bf16 *q, *gate, *k_pages, *v_pages;
    const int *angle, *seq, *pos;
    int ld, angles, rows, Hq, Hk, half;
    float eps;
    PageTable table;
    uint32_t by_page;  // p / page_tokens = p * by_page >> page_shift for p < 2^30, more than any table holds
    int page_shift;
    int per;           // rows of a block
    int* error;
};

constexpr int PREP_THREADS = 256, PREP_ROWS = 128, MANY_ROWS = 512;

__device__ __forceinline__ int page_slot(const PrepArgs& a, int p) { return (int)((uint64_t)(uint32_t)p * a.by_page >> a.page_shift); }
// The page of a place, -1: the table has none.
__device__ __forceinline__ int page_of(const PrepArgs& a, int r, int p) {
    const int sq = a.seq ? a.seq[r] : r, slot = page_slot(a, p);
    if (p < 0 || p >= 1 << 30 || sq < 0 || sq >= a.table.sequences || slot >= a.table.width) return -1;
    return a.table.pages[(size_t)sq * a.table.width + slot];
}

// DH / 8 lanes per head, 8 consecutive dims per lane; the rotary partner of dim d (d +- half) lives half / 8 lanes
// away. A row's units are its Hq query heads, Hk key heads and Hk value heads.
template <int DH>
struct PrepUnit {
    static constexpr int LANES = DH / 8, UNITS = PREP_THREADS / LANES;
    int d0, h;
    bool live, is_q, is_v, writes;  // writes: the block has key or value heads
    __device__ explicit PrepUnit(const PrepArgs& a) {
        const int unit0 = blockIdx.y * UNITS, heads = a.Hq + 2 * a.Hk;
        const int unit = min(unit0 + (int)threadIdx.x / LANES, heads - 1);
        live = unit0 + (int)threadIdx.x / LANES < heads, writes = unit0 + UNITS > a.Hq;
        d0 = threadIdx.x % LANES * 8;
        is_q = unit < a.Hq, is_v = unit >= a.Hq + a.Hk;
        h = is_q ? unit : is_v ? unit - a.Hq - a.Hk : unit - a.Hq;
    }
    __device__ const bf16* row(const PrepArgs& a, int r) const {
        return is_q ? a.qg + (size_t)r * a.ld + (size_t)h * 2 * DH : (is_v ? a.vr : a.kr) + (size_t)r * a.ld + (size_t)h * DH;
    }
    __device__ const bf16* weights(const PrepArgs& a) const { return is_q ? a.qw : a.kw; }
};

template <int DH>
__device__ __forceinline__ void unit_out(const PrepArgs& a, const PrepUnit<DH>& u, int r, uint4 raw, uint4 weight, uint4 gate,
                                         const uint4 (&turns)[2], int page, int off) {
    constexpr int LANES = DH / 8;
    float x[8], wv[8], y[8], cs[8], sn[8];
    unpack8(raw, x);
    unpack8(weight, wv);
    unpack8(turns[0], cs);
    unpack8(turns[1], sn);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss += x[i] * x[i];
    const float inv = rsqrtf(warp_sum<LANES>(ss) / DH + a.eps);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = x[i] * inv * (1.f + wv[i]);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float partner = __shfl_xor_sync(0xffffffffu, x[i], a.half / 8);
        y[i] = x[i];
        if (u.d0 < 2 * a.half) y[i] = x[i] * cs[i] + (u.d0 < a.half ? -partner : partner) * sn[i];
    }
    if (!u.live) return;
    if (u.is_q) {
        st16(a.q + ((size_t)r * a.Hq + u.h) * DH + u.d0, pack8(y));
        st16(a.gate + ((size_t)r * a.Hq + u.h) * DH + u.d0, gate);
    } else if (page >= 0) {
        const size_t at = (((size_t)page * a.table.page_tokens + off) * a.Hk + u.h) * DH + u.d0;
        if (u.is_v)
            st16(a.v_pages + at, raw);
        else
            st16(a.k_pages + at, pack8(y));
    }
}

// Latency bounds it: 251 rows of 16 and 4 heads of 256 (10 MB) take 5.0 us, one row 2.2, launch and all.
template <int DH>
__global__ void __launch_bounds__(PREP_THREADS) attn_prep_paged_kernel(const __grid_constant__ PrepArgs a) {
    grid_dep_trigger();
    grid_dep_sync();
    // A row is a few hundred instructions behind three trips to memory, so whatever does not depend on an
    // earlier trip is asked for at once: row, weights and positions, then page and rotary rows, then the rest.
    const int r = blockIdx.x, tid = threadIdx.x;
    const PrepUnit<DH> u(a);
    const bf16* src = u.row(a, r);
    const uint4 raw = ld16_stream(src + u.d0), weight = ld16(u.weights(a) + u.d0);
    const uint4 gate = u.is_q ? ld16_stream(src + DH + u.d0) : make_uint4(0, 0, 0, 0);
    const int p = a.pos[r], sq = a.seq ? a.seq[r] : r;
    const int turn = a.angle ? a.angle[r] : p;
    const int pt = a.table.page_tokens;
    int pj = u.writes && tid < a.rows ? a.pos[tid] : -1;
    if (p < 0) return;  // the row sits out
    const int slot = page_slot(a, p), off = p - slot * pt;
    int code = 0, page = -1;
    if (p >= 1 << 30 || sq < 0 || sq >= a.table.sequences || slot >= a.table.width)
        code = PAGED_BAD_ROW;
    else if (turn < 0 || turn >= a.angles)
        code = PAGED_BAD_ANGLE;
    else
        page = a.table.pages[(size_t)sq * a.table.width + slot];
    uint4 turns[2] = {};
    if (u.d0 < 2 * a.half && code == 0) {
        // half is a multiple of 8, so the 8 dims of a lane share one aligned table pack
        turns[0] = ld16(a.cos + (size_t)turn * a.half + u.d0 % a.half);
        turns[1] = ld16(a.sin + (size_t)turn * a.half + u.d0 % a.half);
    }
    // Two rows at one place of the cache would race: neither is written.
    bool clash = false;
    for (int j = tid; u.writes && j < a.rows; j += PREP_THREADS) {
        if (j != tid) pj = a.pos[j];
        if (j == r || pj < 0 || pj >= 1 << 30 || pj - page_slot(a, pj) * pt != off) continue;
        const int other = page_of(a, j, pj);
        clash |= other >= 0 && other == page;
    }
    if (code == 0 && (page < 0 || page >= a.table.n_pages)) code = PAGED_BAD_PAGE;
    if (code) {
        if (tid == 0) atomicCAS(a.error, 0, code);
        return;
    }
    if (u.writes && __syncthreads_or(clash)) {
        if (tid == 0) atomicCAS(a.error, 0, PAGED_CLASH);
        page = -1;
    }

    unit_out<DH>(a, u, r, raw, weight, gate, turns, page, off);
}

// Many rows: a block takes `per` of them and looks all others up among these, by a hash of their places in the
// cache; each row against each other by itself took longer than all the rest (8192 rows 223 us, 65536 13.9 ms). The
// next row is asked for while one is worked on. Measured, 24 and 4 heads of 128: 1000 rows 10.4 us (one row a block: 12.9),
// 8192: 69 (223), 65536: 538 (13.9 ms; the bytes alone 287); up to 512 rows one row a block is as quick (6.3 us).
// (rows / 512 of them a block; rows / 1024: 76 and 602, rows / 256: 70 and 538.)
template <int DH>
__global__ void __launch_bounds__(PREP_THREADS) attn_prep_paged_many_kernel(const __grid_constant__ PrepArgs a) {
    constexpr int HASH = 512, AT_ONCE = 4;
    __shared__ int first[HASH], next[PREP_ROWS], places[PREP_ROWS];  // chains of 1 + the row in the block; its place, -1: none
    __shared__ bool clashes[PREP_ROWS];
    grid_dep_trigger();
    grid_dep_sync();
    const PrepUnit<DH> u(a);
    const int tid = threadIdx.x, pt = a.table.page_tokens;
    const int r0 = blockIdx.x * a.per, n = min(a.per, a.rows - r0);
    auto place_of = [&](int r, int p) {
        const int page = page_of(a, r, p);
        return page >= 0 && page < a.table.n_pages ? page * pt + p - page_slot(a, p) * pt : -1;
    };
    auto hash = [](int place) { return (uint32_t)place * 2654435769u >> 23; };
    if (u.writes) {
        for (int i = tid; i < HASH; i += PREP_THREADS) first[i] = 0;
        __syncthreads();
        if (tid < n) {
            places[tid] = place_of(r0 + tid, a.pos[r0 + tid]);
            clashes[tid] = false;
            if (places[tid] >= 0) next[tid] = atomicExch(&first[hash(places[tid])], tid + 1);
        }
        __syncthreads();
        for (int j0 = tid; j0 < a.rows; j0 += AT_ONCE * PREP_THREADS) {
            int place[AT_ONCE];
#pragma unroll
            for (int e = 0; e < AT_ONCE; e++) {
                const int j = min(j0 + e * PREP_THREADS, a.rows - 1);
                place[e] = place_of(j, a.pos[j]);
            }
#pragma unroll
            for (int e = 0; e < AT_ONCE; e++) {
                const int j = min(j0 + e * PREP_THREADS, a.rows - 1);
                if (place[e] < 0) continue;
                for (int i = first[hash(place[e])]; i > 0; i = next[i - 1])
                    if (places[i - 1] == place[e] && r0 + i - 1 != j) clashes[i - 1] = true;
            }
        }
        __syncthreads();
    }
    const uint4 weight = ld16(u.weights(a) + u.d0);
    uint4 raw, gate = make_uint4(0, 0, 0, 0);
    int p;
    auto ask = [&](int r) {
        const bf16* src = u.row(a, r);
        raw = ld16_stream(src + u.d0);
        if (u.is_q) gate = ld16_stream(src + DH + u.d0);
        p = a.pos[r];
    };
    ask(r0);
#pragma unroll 1
    for (int i = 0; i < n; i++) {
        const int r = r0 + i, at = p;
        const uint4 raw_now = raw, gate_now = gate;
        if (i + 1 < n) ask(r + 1);
        if (at < 0) continue;  // sits out
        const int sq = a.seq ? a.seq[r] : r, turn = a.angle ? a.angle[r] : at;
        int code = 0, page = -1;
        uint4 turns[2] = {};
        if (at >= 1 << 30 || sq < 0 || sq >= a.table.sequences || page_slot(a, at) >= a.table.width)
            code = PAGED_BAD_ROW;
        else if (turn < 0 || turn >= a.angles)
            code = PAGED_BAD_ANGLE;
        else {
            page = page_of(a, r, at);
            if (page < 0 || page >= a.table.n_pages) code = PAGED_BAD_PAGE;
            if (u.d0 < 2 * a.half) {
                turns[0] = ld16(a.cos + (size_t)turn * a.half + u.d0 % a.half);
                turns[1] = ld16(a.sin + (size_t)turn * a.half + u.d0 % a.half);
            }
        }
        if (code) {
            if (tid == 0) atomicCAS(a.error, 0, code);
            continue;
        }
        if (u.writes && clashes[i]) {
            if (tid == 0) atomicCAS(a.error, 0, PAGED_CLASH);
            page = -1;
        }
        unit_out<DH>(a, u, r, raw_now, weight, gate_now, turns, page, at - page_slot(a, at) * pt);
    }
}

// ---- attention of one new token per row over its sequence's pages ----
//
// o = sum_t p_t v_t / sum_t p_t, p_t = exp(scale q.k_t - m): one pass with a running maximum and sum.
// Every key and value is read once for all query heads that share it (up to 16 of them, the rows of
// an mma.m16n8k16), which gives at most 16 FLOP per byte: HBM bounds it, not the tensor pipe, and
// tcgen05's 64-row minimum would idle three quarters and more of its rows. So: the copy engine streams
// tiles through a ring of shared memory that holds most of what an SM has, and four warps work on them
// with plain warp-level MMAs.
//
// A tile is HB neighbouring key-value heads (4, 2 or 1) of 16 * 4 / HB tokens: with 4 heads whole rows of
// the pools, or whole kilobytes of them. A warp owns one head's 16 tokens of every tile, its running
// maximum, sum and weighted values stay in its registers, and no warp waits for another until the
// end of a piece, where warps of one head are summed.
//
// Rows of one sequence (a window of new tokens) can share tiles, as many as their heads fit the 16 rows of the
// product: the cache is then read once for them. Where one of them sees tokens of a tile that another does not, the
// product with the values is taken row by row, so that no row gets what lies behind its own length, infinities
// and NaN included. 60 rows in windows of 3, 16 heads over 4 of 128, 20 caches of 8000 tokens (328 MB): 117 -> 64 us.
//
// The work of a launch is one line of tiles (row by row, head block by head block, tokens in order)
// cut into equal runs, one per block, whatever the lengths are. A run's pieces that cover a (row, head
// block) whole are finished by the block; the others leave maximum, sum and weighted values in
// float32 in the workspace, and a second kernel joins the parts of each in order.
//
// Measured, in a recorded graph: 65 caches of 500 to 16000 tokens, 24 query and 4 key-value heads of 128
// (630 MB): 102 us, 6.2 TB/s with the join; 250001 tokens, 16 and 4 heads of 256 (1.02 GB): 160 us, 6.4 TB/s;
// 1500 tokens: 8.3 us; 3 rows of 2 tokens: 7.6. The join takes 5.6, 5.2, 2.9 and 1.5 of these, so the first kernel runs at
// the rate of a copy. Before, tiles of 64 tokens of one head whose warps shared every tile's maximum and probabilities: 119 us (one
// block per SM), 113 (two) for the first.
constexpr int CONSUMERS = 4, PAGED_THREADS = (CONSUMERS + 1) * 32;
constexpr int SLICE = 16;       // tokens of a warp's part of a tile, and of a copied box
constexpr int RUN = 8, PARTS = 64;  // tiles of a run, parts of a piece: see Cut
constexpr int MAX_GROUP = 16;   // query heads of one key-value head that a block takes at once
constexpr int MAX_BLOCKS = 296; // two per SM

template <int DH>
struct PCfg {
    static constexpr int BLOCKS_PER_SM = DH == 128 ? 2 : 1;
    static constexpr int STAGES = 3;
    static constexpr int KV_BYTES = CONSUMERS * SLICE * DH * 2;
    static constexpr int STAGE = 2 * KV_BYTES;
    static constexpr int PART = DH == 128 ? 32 : 64;              // dims that a warp hands over at a time
    static constexpr int PITCH = PART + 4;
    static constexpr int OFF_SUM = STAGES * STAGE;                 // float [4][16][PITCH]
    static constexpr int OFF_ML = OFF_SUM + CONSUMERS * 16 * PITCH * 4;  // float2 [4][16]
    static constexpr int OFF_INV = OFF_ML + CONSUMERS * 16 * 8;    // float [HB][16], 1 / sum
    static constexpr int OFF_BAR = OFF_INV + CONSUMERS * 16 * 4;
    static constexpr int SMEM = OFF_BAR + 2 * STAGES * 8 + 64 + 1024;  // and what aligning the base takes
};

struct PagedArgs {
    const bf16 *q, *gate;
    bf16* out;
    const int *seq, *len;
    float* work;
    int* error;
    int rows, Hq, Hk, group, chunk, chunks;  // group = Hq / Hk in `chunks` parts of at most `chunk` heads
    int window, part;                        // rows that share a block's tiles at most, window * chunk
    uint32_t by_group;                       // m / group = m * by_group >> 16 for m < 16; 0 where window is 1
    int units;                               // chunks * head blocks: what a row's tokens are walked for
    float scale_log2;
    PageTable table;
};
struct PagedMaps {
    CUtensorMap k, v;
};

// Workspace: [blocks][2] parts of [heads][DH] weighted values and [heads] (maximum, sum) pairs, in whole
// 16 bytes (heads = HB * chunk).
// (heads: those of every row that shares the tiles)
__host__ __device__ inline size_t part_floats(int heads, int DH) { return (size_t)heads * DH + (2 * heads + 3) / 4 * 4; }

// PAST_L1: read from L2, for a kernel that runs ahead of the one before it.
template <bool PAST_L1>
__device__ __forceinline__ int load(const int* p) {
    return PAST_L1 ? __ldcg(p) : *p;
}

// Neighbouring rows of one sequence (a causal window) share tiles, up to `window` of them: their heads are rows of
// the same products, each with its own length. A row goes on with the one before it where that one's cache is at most
// SLICE tokens shorter, so that nearly all tiles are whole for both.
// A block finds this out for all rows at once, a bit for each that goes on, in one trip to memory.
constexpr int WINDOW_ROWS = 8192;  // with more rows than this none share
// (lens, if given: the length of every row of a block's THREADS, 0 where it has no tiles)
template <bool PAST_L1, int THREADS>
__device__ __forceinline__ void find_windows(const PagedArgs& a, uint32_t* on, int* lens = nullptr) {
    for (int r0 = threadIdx.x & ~31; r0 < a.rows; r0 += THREADS) {
        const int r = min(r0 + (int)(threadIdx.x & 31), a.rows - 1), b = max(r - 1, 0);
        const int sq = load<PAST_L1>(a.seq + r), sb = load<PAST_L1>(a.seq + b);
        const int n = load<PAST_L1>(a.len + r), nb = load<PAST_L1>(a.len + b);
        const bool has = sq >= 0 && sq < a.table.sequences && n > 0 && n <= a.table.width * a.table.page_tokens;
        const bool goes_on = has && r0 + (int)(threadIdx.x & 31) == r && r > 0 && sq == sb && nb > 0 && n >= nb && n - nb <= SLICE;
        const uint32_t all = __ballot_sync(0xffffffffu, goes_on);
        if (lens && r0 < THREADS) lens[threadIdx.x] = has ? n : 0;
        if ((threadIdx.x & 31) == 0) on[1 + r0 / 32] = all;
    }
    if (threadIdx.x == 0) on[0] = on[1 + (a.rows + 31) / 32] = 0;
    __syncthreads();
}

// How many rows share the tiles of row r; 0: it shares those of a row before it. Counted from the window's first row
// if that is less than LOOK rows before, then from every multiple of `window`, so that no row looks further.
constexpr int LOOK = 32;
__device__ __forceinline__ int rows_from(const PagedArgs& a, const uint32_t* on, int r) {
    const int w = r / 32, bit = r % 32;
    const uint32_t before = __funnelshift_l(on[w], on[w + 1], 31 - bit);          // row r on top, the one before it below
    const uint32_t behind = bit == 31 ? on[w + 2] : __funnelshift_r(on[w + 1], on[w + 2], bit + 1);  // row r + 1 at the bottom
    const int p = __clz(~before);  // rows of the window before r; 32 for as many or more
    int most;
    if (p < LOOK) {
        if (p % a.window) return 0;
        most = min(a.window, LOOK - p);
    } else {
        if (r % a.window && on[(r - LOOK) / 32 + 1] >> (r - LOOK) % 32 & 1) return 0;
        most = a.window - r % a.window;
    }
    return min(most, 1 + __clz(__brev(~behind)));
}

// Tiles of the rows that share those of row r (`together` of them) over all units; 0 for a row that sits out, is empty
// or refused, or shares those of another.
template <bool WINDOWS, bool PAST_L1 = false>
__device__ __forceinline__ long long row_tiles(const PagedArgs& a, const uint32_t* on, int r, int tile, int& tiles, int& together) {
    int n = load<PAST_L1>(a.len + r);
    const int sq = a.seq ? load<PAST_L1>(a.seq + r) : r;
    tiles = 0;
    together = 1;
    if (n <= 0 || sq < 0 || sq >= a.table.sequences || n > (long long)a.table.width * a.table.page_tokens) return 0;
    if constexpr (WINDOWS) {
        together = rows_from(a, on, r);
        if (together == 0) return 0;
        if (together > 1) n = load<PAST_L1>(a.len + r + together - 1);
    }
    tiles = (n + tile - 1) / tile;
    return (long long)tiles * a.units;
}

// The cut of a line of `total` tiles into runs, one per block, none of them empty but those behind the last.
// Runs of one tile as long as the pieces ((row, head block)s, `pieces` of them) come to PARTS parts each on
// average, which the join takes in one trip (16 warps with 4 in flight); from there on runs grow to RUN tiles
// before more parts are made. One row of 24 and 4 heads of 128, a run per block at all lengths and this: 1500
// tokens 8.2 us both, 5000: 12.9 and 10.7, 8000: 14.6 and 12.7, 24000: 20.2 and 17.7, from 38000 on the same.
// (SMs do not stream equally fast: the first block ends some 15 % before the last. Equal runs over three
// quarters and a finer cut of the rest, for whoever is done first, was slower all the same: at 307,000 tokens of 4
// heads 104 -> 107 us as blocks that follow, 118 as blocks that the resident ones take over. A run's start and
// its part cost more than they even out.)
struct Cut {
    long long total;
    int runs;
    __device__ Cut(long long t, int blocks, long long pieces)
        : total(t), runs((int)min((long long)blocks, min(t, max((t + RUN - 1) / RUN, PARTS * pieces)))) {}
    // (up to 2^22 tiles, 67 million tokens, in 32 bits, whose division is shorter)
    __device__ bool small() const { return total < 1 << 22; }
    __device__ long long begin(int r) const { return r >= runs ? total : small() ? (uint32_t)total * r / (uint32_t)runs : total * r / runs; }
    // The last run that begins at or before tile t: floor(total r / runs) <= t just where r <= (runs (t + 1) - 1) / total.
    __device__ int run_of(long long t) const {
        return small() ? (int)(((uint32_t)runs * (uint32_t)(t + 1) - 1) / (uint32_t)total) : (int)((runs * (t + 1) - 1) / total);
    }
};

// Position in the line of tiles.
struct Walk {
    int row, together, unit, tile, tiles;  // unit: head block * chunks + part of the groups
    long long left;
};
template <int TILE, bool WINDOWS>
__device__ __forceinline__ void walk_next_piece(const PagedArgs& a, const uint32_t* on, Walk& w) {
    w.tile = 0;
    if (++w.unit < a.units) return;
    w.unit = 0;
    do {
        w.row++;
    } while (w.row < a.rows && row_tiles<WINDOWS>(a, on, w.row, TILE, w.tiles, w.together) == 0);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two probabilities as two bf16 terms each, hi + lo within 2^-15 of p: hi is p (1 - 2^-16) cut to its upper half,
// which lies below p wherever p > 0, so that lo > 0 too and both products with an infinite value have its sign (with p
// above 2^-117; below, lo may be zero in bf16).
__device__ __forceinline__ void two_terms(float p0, float p1, uint32_t& hi, uint32_t& lo) {
    const uint32_t h0 = __float_as_uint(p0 * 0.9999847412109375f), h1 = __float_as_uint(p1 * 0.9999847412109375f);
    hi = __byte_perm(h0, h1, 0x7632);
    lo = pack2(p0 - __uint_as_float(h0 & 0xffff0000u), p1 - __uint_as_float(h1 & 0xffff0000u));
}
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// The warps of one head meet: all consumers, or the one warp.
template <int SUBS>
__device__ __forceinline__ void piece_sync() {
    if constexpr (SUBS > 1)
        consumer_sync();
    else
        __syncwarp();
}

// (__fdividef is off by 2^-22 at most, and 0 where the divisor passes 2^126)
__device__ __forceinline__ float gated(float o, float gate) { return __fdividef(o, 1.f + __expf(-gate)); }
// Four dims of a result: weighted values times 1 / sum, times the gate's sigmoid, in bf16.
__device__ __forceinline__ uint2 finish4(float4 y, float inv, bool has_gate, uint2 gate) {
    y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
    if (has_gate) {
        y.x = gated(y.x, __uint_as_float(gate.x << 16)), y.y = gated(y.y, __uint_as_float(gate.x & 0xffff0000u));
        y.z = gated(y.z, __uint_as_float(gate.y << 16)), y.w = gated(y.w, __uint_as_float(gate.y & 0xffff0000u));
    }
    return make_uint2(pack2(y.x, y.y), pack2(y.z, y.w));
}

// The second terms of the probabilities are a second product with the values (64 caches of 2000 tokens, 32 heads over one of
// 128: 30.6 us, with one term 27.4), or with at most 8 query heads (FEW) the other 8 rows of the first: as quick as one term.
// (Rows 8 and on of q are loaded as zeros all the same: as constants they made the compiler spill in the loop at
// 256 dims, twice the time.)
template <int DH, int HB, bool WINDOWS, bool FEW>
__global__ void __launch_bounds__(PAGED_THREADS, PCfg<DH>::BLOCKS_PER_SM)
    attn_paged_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ PagedMaps maps) {
    using G = PCfg<DH>;
    constexpr int SUBS = CONSUMERS / HB, TILE = SLICE * SUBS;
    constexpr int BOX_BYTES = HB * SLICE * DH * 2;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::OFF_BAR);
    uint64_t* empty = full + G::STAGES;
    volatile int* gave_up = reinterpret_cast<volatile int*>(empty + G::STAGES);
    __shared__ long long warp_sums[PAGED_THREADS / 32];
    __shared__ Walk begin;
    __shared__ uint32_t on[WINDOWS ? WINDOW_ROWS / 32 + 2 : 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < G::STAGES; s++) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], CONSUMERS);
        }
        *gave_up = 0;
        mbar_init_fence();
        prefetch_tmap(&maps.k);
        prefetch_tmap(&maps.v);
    }
    grid_dep_sync();
    grid_dep_trigger();  // not before: the join reads sequences and lengths without a wait of its own

    // ---- this block's run of the line of tiles ----
    if constexpr (WINDOWS) find_windows<false, PAGED_THREADS>(a, on);
    {
        const int per = (a.rows + PAGED_THREADS - 1) / PAGED_THREADS;
        const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
        long long mine = 0;
        for (int r = r0; r < r1; r++) {
            int tiles, together;
            mine += row_tiles<WINDOWS>(a, on, r, TILE, tiles, together);
        }
        long long upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) warp_sums[warp] = upto;
        __syncthreads();
        long long total = 0;
#pragma unroll
        for (int w = 0; w < PAGED_THREADS / 32; w++) {
            if (w < warp) upto += warp_sums[w];
            total += warp_sums[w];
        }
        const Cut cut(total, gridDim.x, (long long)a.rows * a.units);
        const long long lo = cut.begin(blockIdx.x), hi = cut.begin(blockIdx.x + 1);
        if (tid == 0 && lo == hi) begin.left = 0;
        if (lo < hi && upto - mine <= lo && lo < upto) {
            long long at = upto - mine;
            for (int r = r0; r < r1; r++) {
                int tiles, together;
                const long long n = row_tiles<WINDOWS>(a, on, r, TILE, tiles, together);
                if (lo < at + n) {
                    const int in_row = (int)(lo - at);  // below 2^31: the host limits a row's tiles
                    begin.row = r;
                    begin.together = together;
                    begin.unit = in_row / tiles;
                    begin.tile = in_row % tiles;
                    begin.tiles = tiles;
                    begin.left = hi - lo;
                    break;
                }
                at += n;
            }
        }
        __syncthreads();
    }
    Walk w = begin;
    auto fail = [&](int code) { atomicCAS(a.error, 0, code); };

    if (warp == CONSUMERS) {
        // ---- copies: the whole warp walks, lane b looks up the page of box b and issues its copies ----
        const uint64_t once = policy_evict_first();
        uint32_t it = 0;
        while (w.left > 0) {
            const int n = a.len[w.row + (WINDOWS ? w.together - 1 : 0)], sq = a.seq ? a.seq[w.row] : w.row;
            const int* pages = a.table.pages + (size_t)sq * a.table.width;
            const int column = w.unit / a.chunks * (HB * DH / 64);
            const int from = w.tile;
            const int end = (int)min((long long)w.tiles, w.tile + w.left);
            for (; w.tile < end; w.tile++, w.left--, it++) {
                const int stage = it % G::STAGES;
                const int t = w.tile * TILE + lane * SLICE;
                int at = -1;  // the box's first row in the pools
                if (lane < SUBS && t < n) {
                    const int slot = t / a.table.page_tokens;
                    int page = pages[slot];
                    if (page < 0 || page >= a.table.n_pages) {
                        fail(PAGED_BAD_PAGE);
                        page = 0;
                    }
                    at = page * a.table.page_tokens + (t - slot * a.table.page_tokens);
                }
                if (!mbar_wait(&empty[stage], ((it / G::STAGES) & 1) ^ 1, gave_up)) {
                    fail(PAGED_WAIT);
                    *gave_up = 1;
                    w.left = 0;
                    break;
                }
                const int have = __popc(__ballot_sync(0xffffffffu, at >= 0));
                if (lane == 0) mbar_expect_tx(&full[stage], (uint32_t)have * 2 * BOX_BYTES);
                __syncwarp();
                if (at >= 0) {
                    unsigned char* dst = smem + stage * G::STAGE + lane * BOX_BYTES;
                    tma_load_3d(dst, &maps.k, 0, at, column, &full[stage], once);
                    tma_load_3d(dst + G::KV_BYTES, &maps.v, 0, at, column, &full[stage], once);
                }
            }
            if (w.left > 0) walk_next_piece<TILE, WINDOWS>(a, on, w);
        }
        // rows without tiles: an empty one has nothing to attend to and gets zeros
        for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
            const int n = a.len[r], sq = a.seq ? a.seq[r] : r;
            if (n < 0) continue;
            if (sq < 0 || sq >= a.table.sequences || n > (long long)a.table.width * a.table.page_tokens) {
                if (lane == 0) fail(PAGED_BAD_ROW);
            } else if (n == 0) {
                uint32_t* z = reinterpret_cast<uint32_t*>(a.out + (size_t)r * a.Hq * DH);
                for (int i = lane; i < a.Hq * DH / 2; i += 32) z[i] = 0;
            }
        }
    } else {
        constexpr int NT = DH / 8;                          // n-tiles of 8 dims of the result
        const int mine = warp % HB, sub = warp / HB;        // this warp's head of the block, its slice of the tile
        float* sums = reinterpret_cast<float*>(smem + G::OFF_SUM);
        float2* ml = reinterpret_cast<float2*>(smem + G::OFF_ML);
        float* inverse = reinterpret_cast<float*>(smem + G::OFF_INV);
        const int ra = lane >> 2, rb = ra + 8;              // the two rows (query heads) of this lane's accumulators
        // lane parts of the ldmatrix addresses in the box's tile of 64 dims
        const int k_tok = (lane >> 4) * 8 + (lane & 7), k_ch = (lane >> 3) & 1;
        const int v_tok = lane & 15, v_ch = lane >> 4;
        const uint32_t my_tiles = sub * BOX_BYTES + mine * (DH / 64) * (SLICE * 128);
        // where in q, gate and out the heads of a piece begin, how many rows of the products they are, and where one is
        auto place = [&](const Walk& w, int unit, int& heads) {
            const int h0 = unit % a.chunks * a.chunk;
            heads = WINDOWS ? w.together * a.group : min(a.chunk, a.group - h0);
            return ((size_t)w.row * a.Hq + (size_t)(unit / a.chunks * HB + mine) * a.group + h0) * DH;
        };
        auto of_window = [&](int m) { return WINDOWS ? (int)(m * a.by_group >> 16) : 0; };
        auto head = [&](int m) { return (size_t)(m + of_window(m) * (a.Hq - a.group)) * DH; };
        uint32_t it = 0;
        bool ok = true;
        while (w.left > 0) {
            const int first = a.len[w.row], n = WINDOWS ? a.len[w.row + w.together - 1] : first;  // shortest and longest
            uint32_t qf[DH / 16][4];
            {
                int heads;
                const size_t q_row = place(w, w.unit, heads);
#pragma unroll
                for (int ks = 0; ks < DH / 16; ks++) {
                    const bf16* src = a.q + q_row + ks * 16 + (lane & 3) * 2;
                    qf[ks][0] = ra < heads ? *reinterpret_cast<const uint32_t*>(src + head(ra)) : 0;
                    qf[ks][1] = rb < heads ? *reinterpret_cast<const uint32_t*>(src + head(rb)) : 0;
                    qf[ks][2] = ra < heads ? *reinterpret_cast<const uint32_t*>(src + head(ra) + 8) : 0;
                    qf[ks][3] = rb < heads ? *reinterpret_cast<const uint32_t*>(src + head(rb) + 8) : 0;
                }
            }
            float acc[NT][4] = {};
            float ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
            const int from = w.tile;
            const int end = (int)min((long long)w.tiles, w.tile + w.left);
            for (; w.tile < end; w.tile++, w.left--, it++) {
                const int stage = it % G::STAGES;
                // a warp whose wait ran out waits no more but goes on with the others, which it meets at barriers
                if (ok && !mbar_wait(&full[stage], (it / G::STAGES) & 1, gave_up)) {
                    fail(PAGED_WAIT);
                    *gave_up = 1;
                    ok = false;
                }
                const int left = n - w.tile * TILE - sub * SLICE;  // valid tokens of the slice, from its first on
                if (left > 0) {
                    const uint32_t kb = smem_addr(smem + stage * G::STAGE) + my_tiles, vb = kb + G::KV_BYTES;
                    float s[2][4] = {}, s2[2][4] = {};  // two chains each, so that the products wait less for one another
#pragma unroll
                    for (int ks = 0; ks < DH / 16; ks++) {
                        const int ch = ks * 2 + k_ch;
                        uint32_t b[4];
                        ldsm4(b, kb + (ch >> 3) * (SLICE * 128) + k_tok * 128 + (((ch ^ k_tok) & 7) << 4));
                        mma16816(ks & 1 ? s2[0] : s[0], qf[ks], b[0], b[1]);
                        mma16816(ks & 1 ? s2[1] : s[1], qf[ks], b[2], b[3]);
                    }
                    float xa = -INFINITY, xb = -INFINITY;
                    int left_a = left, left_b = left;
                    const int behind = n - first;  // the shortest row's tokens end that much earlier
                    const bool ragged = WINDOWS && left - behind < SLICE;
                    if (ragged) {
                        left_a -= n - a.len[w.row + min(of_window(ra), w.together - 1)];
                        left_b -= n - a.len[w.row + min(of_window(rb), w.together - 1)];
                    }
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const int token = j * 8 + (lane & 3) * 2 + e;
                            s[j][e] = token < left_a ? (s[j][e] + s2[j][e]) * a.scale_log2 : -INFINITY;
                            xa = fmaxf(xa, s[j][e]);
                            if constexpr (!FEW) {
                                s[j][2 + e] = token < left_b ? (s[j][2 + e] + s2[j][2 + e]) * a.scale_log2 : -INFINITY;
                                xb = fmaxf(xb, s[j][2 + e]);
                            }
                        }
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
                        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, o));
                        if constexpr (!FEW) xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, o));
                    }
                    if (__any_sync(0xffffffffu, xa > ma || xb > mb)) {
                        const float na = fmaxf(ma, xa), nb = fmaxf(mb, xb);
                        const float fa = ma == -INFINITY ? 0.f : exp2f(ma - na), fb = FEW ? fa : mb == -INFINITY ? 0.f : exp2f(mb - nb);
                        ma = na, mb = nb;
                        la *= fa, lb *= fb;
#pragma unroll
                        for (int t = 0; t < NT; t++) acc[t][0] *= fa, acc[t][1] *= fa, acc[t][2] *= fb, acc[t][3] *= fb;
                    }
                    // a row without a finite score so far keeps offset 0: its terms are exp2(-inf) = 0
                    const float oa = ma == -INFINITY ? 0.f : ma, ob = mb == -INFINITY ? 0.f : mb;
                    uint32_t pf[4], pr[4];
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float p0 = exp2f(s[j][0] - oa), p1 = exp2f(s[j][1] - oa);
                        la += p0 + p1;
                        if constexpr (FEW) {
                            two_terms(p0, p1, pf[2 * j], pf[2 * j + 1]);
                        } else {
                            const float p2 = exp2f(s[j][2] - ob), p3 = exp2f(s[j][3] - ob);
                            lb += p2 + p3;
                            two_terms(p0, p1, pf[2 * j], pr[2 * j]);
                            two_terms(p2, p3, pf[2 * j + 1], pr[2 * j + 1]);
                        }
                    }
                    // values behind the last token may be anything, NaN included: their products with a
                    // probability of zero have to be zero
                    auto kept = [&](int tokens, int e) {
                        const int t0 = e * 8 + (lane & 3) * 2;
                        return (t0 < tokens ? 0xffffu : 0u) | (t0 + 1 < tokens ? 0xffff0000u : 0u);
                    };
                    if (!ragged || behind == 0) {
                        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
                        if (left < SLICE) keep[0] = kept(left, 0), keep[1] = kept(left, 1);
#pragma unroll
                        for (int t = 0; t < NT; t += 4) {
                            uint32_t b[2][4];
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const int ch = v_ch + t + 2 * u;
                                ldsm4_t(b[u], vb + (ch >> 3) * (SLICE * 128) + v_tok * 128 + (((ch ^ v_tok) & 7) << 4));
#pragma unroll
                                for (int e = 0; e < 4; e++) b[u][e] &= keep[e & 1];
                            }
#pragma unroll
                            for (int u = 0; u < 4; u++) mma16816(acc[t + u], pf, b[u / 2][u % 2 * 2], b[u / 2][u % 2 * 2 + 1]);
                            if constexpr (!FEW) {
#pragma unroll
                                for (int u = 0; u < 4; u++) mma16816(acc[t + u], pr, b[u / 2][u % 2 * 2], b[u / 2][u % 2 * 2 + 1]);
                            }
                        }
                    } else {
                        // a token that one row of the window has and another has not: each row on its own
#pragma unroll 1
                        for (int i = 0; i < w.together; i++) {
                            const int tokens = left - (n - a.len[w.row + i]);
                            if (tokens <= 0) continue;
                            const bool is_a = of_window(ra) == i, is_b = of_window(rb) == i;
                            const uint32_t keep[2] = {kept(tokens, 0), kept(tokens, 1)};
                            const uint32_t own[4] = {is_a ? pf[0] : 0, is_b ? pf[1] : 0, is_a ? pf[2] : 0, is_b ? pf[3] : 0};
                            const uint32_t rest[4] = {is_a ? pr[0] : 0, is_b ? pr[1] : 0, is_a ? pr[2] : 0, is_b ? pr[3] : 0};
#pragma unroll
                            for (int t = 0; t < NT; t += 2) {
                                const int ch = v_ch + t;
                                uint32_t b[4];
                                ldsm4_t(b, vb + (ch >> 3) * (SLICE * 128) + v_tok * 128 + (((ch ^ v_tok) & 7) << 4));
#pragma unroll
                                for (int u = 0; u < 2; u++) {
                                    float x[4] = {acc[t + u][0], acc[t + u][1], acc[t + u][2], acc[t + u][3]};
                                    mma16816(x, rest, b[2 * u] & keep[0], b[2 * u + 1] & keep[1]);
                                    mma16816(x, own, b[2 * u] & keep[0], b[2 * u + 1] & keep[1]);
                                    if (is_a) acc[t + u][0] = x[0], acc[t + u][1] = x[1];
                                    if (is_b) acc[t + u][2] = x[2], acc[t + u][3] = x[3];
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
            }

            // ---- the piece's end ----
            if constexpr (FEW) {
#pragma unroll
                for (int t = 0; t < NT; t++) acc[t][0] += acc[t][2], acc[t][1] += acc[t][3];
            }
            // The warps hand their weighted values over in shared memory, some dims at a time, and those of a head
            // sum, norm and write them. One loop for it, the accumulators moving up: unrolled, the code took longer to
            // fetch than to run, and every gate waited for the store before it (5 us a piece at 128 dims, 17 at 256).
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                la += __shfl_xor_sync(0xffffffffu, la, o);
                lb += __shfl_xor_sync(0xffffffffu, lb, o);
            }
            // Places are computed again from what the compiler takes for new values: held in registers through the
            // loop they would spill some of its own.
            int unit = w.unit, heads, own = threadIdx.x;
            asm volatile("" : "+r"(unit), "+r"(own));
            const size_t q_row = place(w, unit, heads);
            const int lane = own & 31, warp = own >> 5, mine = warp % HB, sub = warp / HB, ra = lane >> 2, rb = ra + 8;
            const bool whole = from == 0 && end == w.tiles;
            // the part that begins a (row, unit) lies in place 1, one that continues it in place 0
            float* const part_at = a.work + ((size_t)blockIdx.x * 2 + (from == 0 ? 1 : 0)) * part_floats(HB * a.part, DH);
            float2* const pairs_at = reinterpret_cast<float2*>(part_at + (size_t)HB * a.part * DH) + mine * a.part;
            if (SUBS == 1 && !whole) {  // nothing to sum or to gate
                float* val = part_at + (size_t)mine * a.part * DH + (lane & 3) * 2;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if (ra < heads) *reinterpret_cast<float2*>(val + ra * DH + t * 8) = make_float2(acc[t][0], acc[t][1]);
                    if (rb < heads) *reinterpret_cast<float2*>(val + rb * DH + t * 8) = make_float2(acc[t][2], acc[t][3]);
                }
                if ((lane & 3) == 0 && ra < heads) pairs_at[ra] = make_float2(ma, la);
                if ((lane & 3) == 0 && rb < heads) pairs_at[rb] = make_float2(mb, lb);
                if (w.left > 0) walk_next_piece<TILE, WINDOWS>(a, on, w);
                continue;
            }
            if ((lane & 3) == 0) ml[warp * 16 + ra] = make_float2(ma, la), ml[warp * 16 + rb] = make_float2(mb, lb);
            piece_sync<SUBS>();
            auto joined = [&](int row) {  // maximum and sum of a row over the warps of the head
                float m = -INFINITY, l = 0.f;
#pragma unroll
                for (int u = 0; u < SUBS; u++) m = fmaxf(m, ml[(u * HB + mine) * 16 + row].x);
#pragma unroll
                for (int u = 0; u < SUBS; u++) {
                    const float2 x = ml[(u * HB + mine) * 16 + row];
                    l += x.y * exp2f(x.x - (m == -INFINITY ? 0.f : m));
                }
                return make_float2(m, l);
            };
            float fa = 1.f, fb = 1.f;
            if constexpr (SUBS > 1) {
                const float na = joined(ra).x, nb = joined(rb).x;
                fa = exp2f(ma - (na == -INFINITY ? 0.f : na)), fb = exp2f(mb - (nb == -INFINITY ? 0.f : nb));
            }
            if (sub == 0 && lane < heads) {
                const float2 x = joined(lane);
                if (whole)
                    inverse[mine * 16 + lane] = x.y == 0.f ? 0.f : 1.f / x.y;
                else
                    pairs_at[lane] = x;
            }
            constexpr int QUADS = G::PART / 4, STEPS = 16 * QUADS / (32 * SUBS);  // fours of dims, and how many of them a lane writes
            float* const box = sums + warp * 16 * G::PITCH;
            uint2 gate[STEPS];
            auto gates = [&](int d0) {
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    const int at = (i * SUBS + sub) * 32 + lane, row = at / QUADS;
                    if (a.gate && whole && row < heads)
                        gate[i] = __ldg(reinterpret_cast<const uint2*>(a.gate + q_row + head(row) + d0 + at % QUADS * 4));
                }
            };
            gates(0);
#pragma unroll 1
            for (int d0 = 0; d0 < DH; d0 += G::PART) {
#pragma unroll
                for (int t = 0; t < G::PART / 8; t++) {
                    const int d = t * 8 + (lane & 3) * 2;
                    *reinterpret_cast<float2*>(box + ra * G::PITCH + d) = make_float2(acc[t][0] * fa, acc[t][1] * fa);
                    if constexpr (!FEW) *reinterpret_cast<float2*>(box + rb * G::PITCH + d) = make_float2(acc[t][2] * fb, acc[t][3] * fb);
                }
                piece_sync<SUBS>();
#pragma unroll
                for (int i = 0; i < STEPS; i++) {
                    const int at = (i * SUBS + sub) * 32 + lane, row = at / QUADS, d = at % QUADS * 4;
                    if (row >= heads) continue;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int u = 0; u < SUBS; u++) {
                        const float4 x = *reinterpret_cast<const float4*>(sums + ((u * HB + mine) * 16 + row) * G::PITCH + d);
                        y.x += x.x, y.y += x.y, y.z += x.z, y.w += x.w;
                    }
                    if (whole) {
                        *reinterpret_cast<uint2*>(a.out + q_row + head(row) + d0 + d) =
                            finish4(y, inverse[mine * 16 + row], a.gate != nullptr, gate[i]);
                    } else {
                        *reinterpret_cast<float4*>(part_at + ((size_t)mine * a.part + row) * DH + d0 + d) = y;
                    }
                }
                if (d0 + G::PART < DH) gates(d0 + G::PART);
                piece_sync<SUBS>();
#pragma unroll
                for (int t = 0; t < NT - G::PART / 8; t++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[t][e] = acc[t + G::PART / 8][e];
            }
            if (w.left > 0) walk_next_piece<TILE, WINDOWS>(a, on, w);
        }
    }
    // after an abort give copies in flight time to land before the shared memory is released
    if (*gave_up) __nanosleep(1000000);
    __syncthreads();
}

// Joins the parts of the (row, unit)s that were cut. One begins in some run of the first kernel (place 1 of
// its block's parts) and goes on in the runs after it (their place 0). Which these are follows from the
// lengths, so every block finds them out while the first kernel still runs, and waits for that only to read
// the parts (1500 tokens 9.0 -> 8.2 us, against notes that the first kernel left). The items are the query heads
// of these; a warp takes one at a time, or a whole block where items are few. The order of the sums is fixed by
// the cut alone. What follows the wait is a chain of trips to L2, so the code is kept short: unrolled further it
// took longer to fetch than to run. (Held to 64 registers it was 2 us slower in large calls; blocks that take 32 dims
// of an item with four parts to a warp, so that few items keep all blocks busy, cost 1 to 4 us more.)
constexpr int JOIN_WARPS = 16, JOIN_BLOCKS = 148;

template <int DH, bool WINDOWS>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attn_paged_join_kernel(const __grid_constant__ PagedArgs a, int blocks, int HB) {
    constexpr int E = DH / 128, U = 4, THREADS = JOIN_WARPS * 32;  // U: parts in flight per warp
    __shared__ int4 cuts[MAX_BLOCKS];  // row, unit, first run, last run
    __shared__ int base[JOIN_WARPS], cut_rows[MAX_BLOCKS], widest;
    __shared__ long long upto[THREADS], warp_sums[JOIN_WARPS];
    __shared__ __align__(16) float sums[JOIN_WARPS][DH];
    __shared__ float2 pairs[JOIN_WARPS];
    __shared__ uint32_t on[WINDOWS ? WINDOW_ROWS / 32 + 2 : 1];
    __shared__ int lens[WINDOWS ? THREADS : 1];
    grid_dep_trigger();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tile = SLICE * CONSUMERS / HB;
    const size_t floats = part_floats(HB * a.part, DH);
    if (tid == 0) widest = 1;
    if constexpr (WINDOWS) find_windows<true, THREADS>(a, on, lens);
    // tiles up to the end of every thread's rows
    const int per = (a.rows + THREADS - 1) / THREADS;
    int most = 0;
    {
        long long mine = 0;
        for (int r = min(tid * per, a.rows), end = min(r + per, a.rows); r < end; r++) {
            int tiles = 0, together;
            if (WINDOWS && per == 1) {  // without another trip
                together = lens[r] > 0 ? rows_from(a, on, r) : 0;
                if (together > 0) tiles = (lens[r + together - 1] + tile - 1) / tile;
                mine = (long long)tiles * a.units;
            } else {
                mine += row_tiles<WINDOWS, true>(a, on, r, tile, tiles, together);
            }
            most = max(most, tiles);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, mine, o);
            if (lane >= o) mine += x;
        }
        if (lane == 31) warp_sums[warp] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; w++)
            if (w < warp) mine += warp_sums[w];
        upto[tid] = mine;
        __syncthreads();
    }
    const Cut cut(upto[THREADS - 1], blocks, (long long)a.rows * a.units);
    // thread b: whether run b ends within a (row, unit) that begins in it; their list
    int count = 0;
    // (runs and rows of one tile each: none)
    if (__syncthreads_or(most > 1 || cut.runs < cut.total)) {
        int4 found = make_int4(-1, 0, 0, 0);
        int found_rows = 1;
        if (tid < cut.runs - 1) {
            const long long t = cut.begin(tid + 1);
            int c = 0;  // the thread whose rows hold tile t
            for (int step = 1 << (31 - __clz((a.rows + per - 1) / per)); step; step /= 2)
                if (upto[c + step - 1] <= t) c += step;
            long long at = c ? upto[c - 1] : 0;
            for (int r = c * per; r < a.rows; r++) {
                int tiles, together = 1;
                long long n;
                if (per == 1)
                    n = upto[c] - at, tiles = (int)n / a.units, together = WINDOWS ? rows_from(a, on, r) : 1;
                else
                    n = row_tiles<WINDOWS, true>(a, on, r, tile, tiles, together);
                if (at + n <= t) {
                    at += n;
                    continue;
                }
                const int in_row = (int)(t - at), of = in_row % tiles;
                if (of > 0 && t - of >= cut.begin(tid)) {
                    found = make_int4(r, in_row / tiles, tid, cut.run_of(t - of + tiles - 1));
                    found_rows = together;
                }
                break;
            }
        }
        const uint32_t all = __ballot_sync(0xffffffffu, found.x >= 0);
        if (lane == 0) base[warp] = __popc(all);
        __syncthreads();
        int at = __popc(all & ((1u << lane) - 1));
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; w++) {
            if (w < warp) at += base[w];
            count += base[w];
        }
        if (found.x >= 0) {
            cuts[at] = found;
            if (WINDOWS) cut_rows[at] = found_rows, atomicMax(&widest, found_rows);
        }
        __syncthreads();
    }
    grid_dep_sync();
    const int rows = WINDOWS ? widest * a.group : a.chunk, heads = HB * rows;  // of the products, as many as any has
    const int items = count * heads;
    const bool together = items <= 2 * (int)gridDim.x;
    const int width = together ? 1 : JOIN_WARPS;
    for (int item = blockIdx.x * width + (together ? 0 : warp); item < items; item += gridDim.x * width) {
        const int4 piece = cuts[item / heads];
        const int of = item % heads / rows, i = item % rows, slot = of * a.part + i;
        const int hk = piece.y / a.chunks * HB + of, h0 = piece.y % a.chunks * a.chunk;
        if (i >= (WINDOWS ? cut_rows[item / heads] * a.group : min(a.chunk, a.group - h0))) continue;
        const int of_window = WINDOWS ? (int)(i * a.by_group >> 16) : 0;
        const size_t at = ((size_t)(piece.x + of_window) * a.Hq + (size_t)hk * a.group + h0 + i - of_window * a.group) * DH;
        float m = -INFINITY, l = 0.f;
        float4 acc[E] = {};
        uint2 gate[E] = {};
        if (a.gate && (!together || warp == 0)) {
#pragma unroll
            for (int e = 0; e < E; e++) gate[e] = __ldg(reinterpret_cast<const uint2*>(a.gate + at + e * 128 + lane * 4));
        }
        const int stride = together ? JOIN_WARPS : 1;
        for (int p0 = piece.z + (together ? warp : 0); p0 <= piece.w; p0 += U * stride) {
            float2 ml[U];
            float4 x[U][E];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int p = p0 + u * stride;
                ml[u] = make_float2(-INFINITY, 0.f);
                if (p <= piece.w) {
                    const float* part = a.work + ((size_t)p * 2 + (p == piece.z)) * floats;
                    ml[u] = reinterpret_cast<const float2*>(part + (size_t)HB * a.part * DH)[slot];
#pragma unroll
                    for (int e = 0; e < E; e++) x[u][e] = *reinterpret_cast<const float4*>(part + (size_t)slot * DH + e * 128 + lane * 4);
                }
            }
            float mm = m;
#pragma unroll
            for (int u = 0; u < U; u++) mm = fmaxf(mm, ml[u].x);
            const float off = mm == -INFINITY ? 0.f : mm, f = exp2f(m - off);
            m = mm, l *= f;
#pragma unroll
            for (int e = 0; e < E; e++) acc[e].x *= f, acc[e].y *= f, acc[e].z *= f, acc[e].w *= f;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (p0 + u * stride <= piece.w) {
                    const float c = exp2f(ml[u].x - off);
                    l += ml[u].y * c;
#pragma unroll
                    for (int e = 0; e < E; e++)
                        acc[e].x += c * x[u][e].x, acc[e].y += c * x[u][e].y, acc[e].z += c * x[u][e].z, acc[e].w += c * x[u][e].w;
                }
        }
        if (together) {
#pragma unroll
            for (int e = 0; e < E; e++) *reinterpret_cast<float4*>(&sums[warp][e * 128 + lane * 4]) = acc[e];
            if (lane == 0) pairs[warp] = make_float2(m, l);
            __syncthreads();
            m = -INFINITY;
            for (int w = 0; w < JOIN_WARPS; w++) m = fmaxf(m, pairs[w].x);
            const float off = m == -INFINITY ? 0.f : m;
            l = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (warp == 0)
                for (int w = 0; w < JOIN_WARPS; w++) {
                    const float c = exp2f(pairs[w].x - off);
                    l += pairs[w].y * c;
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float4 x = *reinterpret_cast<const float4*>(&sums[w][e * 128 + lane * 4]);
                        acc[e].x += c * x.x, acc[e].y += c * x.y, acc[e].z += c * x.z, acc[e].w += c * x.w;
                    }
                }
            __syncthreads();
        }
        if (together && warp > 0) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const size_t d = at + e * 128 + lane * 4;
            *reinterpret_cast<uint2*>(a.out + d) = finish4(acc[e], inv, a.gate != nullptr, gate[e]);
        }
    }
}

// The attention step operators' error word on the current device, looked up once per device.
int error_word(int** p, int* device) {
    static int* address[64] = {};
    const cudaError_t e = cudaGetDevice(device);
    if (e != cudaSuccess) return e;
    if (*device >= 64) return cudaErrorInvalidDevice;
    if (!address[*device]) {
        int* a = nullptr;
        const int rc = step_error_address(STEP_ATTENTION, &a);
        if (rc != 0) return rc;
        address[*device] = a;
    }
    *p = address[*device];
    return 0;
}

bool table_ok(const PageTable& t) {
    return t.pages && t.width > 0 && t.sequences > 0 && t.n_pages > 0 && t.page_tokens > 0 &&
           (long long)t.n_pages * t.page_tokens <= 0x7fffffffLL && (long long)t.width * t.page_tokens <= (1LL << 30);
}

// Key-value heads of a tile: as many as share the pool's rows, up to a warp each.
inline int head_block(int Hk) { return Hk % 4 == 0 ? 4 : Hk % 2 == 0 ? 2 : 1; }

template <int DH, int HB, bool WINDOWS, bool FEW>
int run_paged(const PagedArgs& a, const PagedMaps& maps, int dev, int blocks, cudaStream_t st) {
    using G = PCfg<DH>;
    static bool configured[64] = {};
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(attn_paged_kernel<DH, HB, WINDOWS, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaError_t e = launch_dep_family(DEP_ATTENTION, attn_paged_kernel<DH, HB, WINDOWS, FEW>, blocks, PAGED_THREADS, G::SMEM, st, a, maps);
    if (e != cudaSuccess) return e;
    // always a programmatic dependent: it waits for the first kernel before it reads anything of it
    e = launch_maybe_dep(true, attn_paged_join_kernel<DH, WINDOWS>, JOIN_BLOCKS, JOIN_WARPS * 32, 0, st, a, blocks, HB);
    return e != cudaSuccess ? e : cudaGetLastError();
}

template <int DH, bool WINDOWS, bool FEW>
int run_paged(int HB, const PagedArgs& a, const PagedMaps& maps, int dev, int blocks, cudaStream_t st) {
    return HB == 4   ? run_paged<DH, 4, WINDOWS, FEW>(a, maps, dev, blocks, st)
           : HB == 2 ? run_paged<DH, 2, WINDOWS, FEW>(a, maps, dev, blocks, st)
                     : run_paged<DH, 1, WINDOWS, FEW>(a, maps, dev, blocks, st);
}

// Blocks of a call at most: what its workspace is for.
inline int most_blocks(int Dh) { return Dh == 256 ? MAX_BLOCKS / 2 * PCfg<256>::BLOCKS_PER_SM : MAX_BLOCKS / 2 * PCfg<128>::BLOCKS_PER_SM; }

// How a key-value head's query heads go into blocks, and how many rows of a sequence may share the 16 rows of a product.
struct Heads {
    int group, chunks, chunk, window;
    Heads(int Hq, int Hk)
        : group(Hq / Hk), chunks((group + MAX_GROUP - 1) / MAX_GROUP), chunk((group + chunks - 1) / chunks),
          window(chunks == 1 ? MAX_GROUP / group : 1) {}
};

}  // namespace
}  // namespace s1

using namespace s1;

extern "C" int s1_attn_prep_paged(const void* qg, const void* kr, const void* vr, int ld, const void* qw, const void* kw,
                                  const void* cos, const void* sin, int angles, const int* angle, void* q, void* gate,
                                  void* k_pages, void* v_pages, int n_pages, int page_tokens, const int* table,
                                  int table_pages, int n_seqs, const int* seq, const int* pos, int rows, int Hq, int Hk,
                                  int Dh, int half, float eps, void* stream) {
    if ((Dh != 128 && Dh != 256) || Hq <= 0 || Hk <= 0 || Hq > (1 << 20) || Hk > (1 << 20) || rows < 0 || rows > 65536 || angles < 0 || ld % 8 != 0 ||
        ld < 2LL * Hq * Dh || ld < (long long)Hk * Dh)
        return cudaErrorInvalidValue;
    // the lane ^ (half / 8) partner exchange needs half a multiple of 8, half / 8 a power of two, 2 * half <= Dh
    if (half <= 0 || half % 8 != 0 || 2 * half > Dh || ((half / 8) & (half / 8 - 1))) return cudaErrorInvalidValue;
    if (rows == 0) return cudaSuccess;
    const PageTable t{table, table_pages, n_seqs, n_pages, page_tokens};
    if (!table_ok(t) || !pos) return cudaErrorInvalidValue;
    for (const void* p : {qg, kr, vr, qw, kw, cos, sin, (const void*)q, (const void*)gate, (const void*)k_pages, (const void*)v_pages})
        if (!p || !aligned16(p)) return cudaErrorInvalidValue;
    PrepArgs a{};
    a.qg = static_cast<const bf16*>(qg), a.kr = static_cast<const bf16*>(kr), a.vr = static_cast<const bf16*>(vr);
    a.qw = static_cast<const bf16*>(qw), a.kw = static_cast<const bf16*>(kw);
    a.cos = static_cast<const bf16*>(cos), a.sin = static_cast<const bf16*>(sin);
    a.q = static_cast<bf16*>(q), a.gate = static_cast<bf16*>(gate);
    a.k_pages = static_cast<bf16*>(k_pages), a.v_pages = static_cast<bf16*>(v_pages);
    a.angle = angle, a.seq = seq, a.pos = pos;
    a.ld = ld, a.angles = angles, a.rows = rows, a.Hq = Hq, a.Hk = Hk, a.half = half, a.eps = eps, a.table = t;
    int shift = 31 - __builtin_clz(page_tokens);
    a.page_shift = 31 + shift, a.by_page = (uint32_t)((1ULL << a.page_shift) / page_tokens + 1);
    a.per = rows <= MANY_ROWS ? 1 : std::max(2, std::min(PREP_ROWS, rows / 512));
    const int units = PREP_THREADS / (Dh / 8);
    const dim3 grid((rows + a.per - 1) / a.per, (Hq + 2 * Hk + units - 1) / units);
    if (grid.y > 65535) return cudaErrorInvalidValue;
    int dev = 0;
    const int rc = error_word(&a.error, &dev);
    if (rc != 0) return rc;
    auto* const one = Dh == 256 ? attn_prep_paged_kernel<256> : attn_prep_paged_kernel<128>;
    auto* const many = Dh == 256 ? attn_prep_paged_many_kernel<256> : attn_prep_paged_many_kernel<128>;
    const cudaError_t e = launch_dep(a.per == 1 ? one : many, grid, PREP_THREADS, 0, as_stream(stream), a);
    return e != cudaSuccess ? e : cudaGetLastError();
}

extern "C" size_t s1_attention_paged_workspace_floats(int Hq, int Hk, int Dh) {
    if (Hq <= 0 || Hk <= 0 || Hq % Hk != 0 || (Dh != 128 && Dh != 256)) return 0;
    const Heads h(Hq, Hk);
    return (size_t)most_blocks(Dh) * 2 * part_floats(head_block(Hk) * h.window * h.chunk, Dh);
}

extern "C" int s1_attention_paged(const void* q, const void* gate, void* out, const void* k_pages, const void* v_pages,
                                  int n_pages, int page_tokens, const int* table, int table_pages, int n_seqs, const int* seq,
                                  const int* len, int rows, int Hq, int Hk, int Dh, float scale, float* workspace,
                                  size_t workspace_floats, void* stream) {
    if ((Dh != 128 && Dh != 256) || Hk <= 0 || Hq <= 0 || Hq % Hk != 0 || rows < 0 || rows > (1 << 20) || page_tokens <= 0 ||
        page_tokens % 16 != 0)
        return cudaErrorInvalidValue;
    if (rows == 0) return cudaSuccess;
    const PageTable t{table, table_pages, n_seqs, n_pages, page_tokens};
    if (!table_ok(t) || !q || !out || !k_pages || !v_pages || !len || !workspace) return cudaErrorInvalidValue;
    if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(workspace) || !aligned16(q) || !aligned16(out) || !aligned16(gate))
        return cudaErrorInvalidValue;
    if (workspace_floats < s1_attention_paged_workspace_floats(Hq, Hk, Dh)) return cudaErrorInvalidValue;
    PagedArgs a{};
    const Heads h(Hq, Hk);
    a.group = h.group, a.chunks = h.chunks, a.chunk = h.chunk, a.window = h.window, a.part = h.window * h.chunk;
    a.by_group = a.window > 1 ? 65536 / a.group + 1 : 0;
    const int HB = head_block(Hk), tile = SLICE * CONSUMERS / HB;
    if ((long long)(Hk / HB) * a.chunks > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.units = Hk / HB * a.chunks;
    const long long row_most = ((long long)table_pages * page_tokens + tile - 1) / tile * a.units;
    if (row_most > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.q = static_cast<const bf16*>(q), a.gate = static_cast<const bf16*>(gate), a.out = static_cast<bf16*>(out);
    a.seq = seq, a.len = len, a.work = workspace, a.rows = rows, a.Hq = Hq, a.Hk = Hk, a.table = t;
    a.scale_log2 = scale * 1.4426950408889634f;
    int dev = 0;
    const int rc = error_word(&a.error, &dev);
    if (rc != 0) return rc;
    static int sm_count[64] = {};
    if (!sm_count[dev]) {
        const cudaError_t e = cudaDeviceGetAttribute(&sm_count[dev], cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
    }
    PagedMaps maps;
    const uint64_t pool_rows = (uint64_t)n_pages * page_tokens, width = (uint64_t)Hk * Dh;
    if (!tensor_map_columns(k_pages, pool_rows, width, SLICE, HB * Dh, &maps.k) ||
        !tensor_map_columns(v_pages, pool_rows, width, SLICE, HB * Dh, &maps.v))
        return CS1_ERR_TENSOR_MAP;
    const int per_sm = Dh == 256 ? PCfg<256>::BLOCKS_PER_SM : PCfg<128>::BLOCKS_PER_SM;
    const int blocks = (int)std::min<long long>(std::min(most_blocks(Dh), sm_count[dev] * per_sm), rows * row_most);
    const cudaStream_t st = as_stream(stream);
    // Whether rows may share tiles: it costs some 2 us in lookups, so not where there are no windows (no more rows than
    // sequences), nor where L2 is quick enough with what rows of one sequence read again, the more so the fewer of
    // them share. Windows of 3 rows, each alone and shared: 16 heads over 4, caches of 16 MB 13.2 and 15.6 us, 33 MB
    // 21.7 and 20.3, 330 MB 117 and 64; 24 over 4 (two of the rows share), 33 MB 20.4 and 22.5, 66 MB 39.0 and 34.0,
    // 120 MB 62 and 37.
    const double bytes = (double)n_seqs * table_pages * page_tokens * Hk * Dh * 4;
    const bool windows = seq && rows > n_seqs && rows <= WINDOW_ROWS && bytes * (a.window - 1) >= 64e6;
    if (windows)
        return Dh == 256 ? run_paged<256, true, false>(HB, a, maps, dev, blocks, st) : run_paged<128, true, false>(HB, a, maps, dev, blocks, st);
    // Few heads, the second terms in the idle rows against a second product: 8000 tokens of 24 and 4 heads 12.3 us and 14.4, 32 x
    // 32,000 313 and 325, 250001 tokens of 16 and 4 heads of 256, called for seconds on end, 162 and 167.
    if (a.chunk <= 8)
        return Dh == 256 ? run_paged<256, false, true>(HB, a, maps, dev, blocks, st) : run_paged<128, false, true>(HB, a, maps, dev, blocks, st);
    return Dh == 256 ? run_paged<256, false, false>(HB, a, maps, dev, blocks, st) : run_paged<128, false, false>(HB, a, maps, dev, blocks, st);
}
