// Full attention of the tokens after a prefill, over a cache kept in pages: norm, rotary and gate split
// of new rows with their keys and values put into the cache, and the attention of new rows over it.
//
// A cache is two pools [n_pages, page_tokens, Hk, Dh] (keys after norm and rotary, values as
// projected) and a table [sequences, table_pages] of page numbers: token p of a sequence is row
// p % page_tokens of page table[p / page_tokens]. Several sequences may name the same page.
//
// Float32 from the inputs to one rounding at the end (the prefill's operators round in between where
// the model stores a tensor, so bf16 results may differ from theirs by a step); only the probabilities
// are rounded to bf16 on their way into the product with the values, as in the prefill's attention.
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

// Codes left in the attention family's device error word.
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
    int* error;
};

constexpr int PREP_THREADS = 256;

// DH / 8 lanes per head, 8 consecutive dims per lane; the rotary partner of dim d (d +- half) lives
// half / 8 lanes away. A row's units are its Hq query heads, Hk key heads and Hk value heads.
template <int DH>
__global__ void __launch_bounds__(PREP_THREADS) attn_prep_paged_kernel(const __grid_constant__ PrepArgs a) {
    constexpr int LANES = DH / 8, UNITS = PREP_THREADS / LANES;
    grid_dep_trigger();
    grid_dep_sync();
    const int r = blockIdx.x, tid = threadIdx.x;
    const int p = a.pos[r], sq = a.seq ? a.seq[r] : r;
    if (p < 0) return;  // the row sits out
    const int turn = a.angle ? a.angle[r] : p;
    const int slot = p / a.table.page_tokens, off = p - slot * a.table.page_tokens;
    int code = 0, page = -1;
    if (sq < 0 || sq >= a.table.sequences || slot >= a.table.width)
        code = PAGED_BAD_ROW;
    else if (turn < 0 || turn >= a.angles)
        code = PAGED_BAD_ANGLE;
    else {
        page = a.table.pages[(size_t)sq * a.table.width + slot];
        if (page < 0 || page >= a.table.n_pages) code = PAGED_BAD_PAGE;
    }
    if (code) {
        if (tid == 0) atomicCAS(a.error, 0, code);
        return;
    }
    const int unit0 = blockIdx.y * UNITS;
    const int heads = a.Hq + 2 * a.Hk;
    const int unit = min(unit0 + tid / LANES, heads - 1);
    const bool live = unit0 + tid / LANES < heads;
    const int d0 = tid % LANES * 8;
    const bool is_q = unit < a.Hq, is_v = unit >= a.Hq + a.Hk;
    const int h = is_q ? unit : is_v ? unit - a.Hq - a.Hk : unit - a.Hq;
    const bf16* src = is_q ? a.qg + (size_t)r * a.ld + (size_t)h * 2 * DH : (is_v ? a.vr : a.kr) + (size_t)r * a.ld + (size_t)h * DH;
    const uint4 raw = ld16_stream(src + d0);

    // Two rows at one place of the cache would race: neither is written.
    if (unit0 + UNITS > a.Hq) {
        bool clash = false;
        for (int j = tid; j < a.rows; j += PREP_THREADS) {
            const int pj = a.pos[j];
            if (j == r || pj < 0 || pj % a.table.page_tokens != off) continue;
            const int sj = a.seq ? a.seq[j] : j, slot_j = pj / a.table.page_tokens;
            if (sj < 0 || sj >= a.table.sequences || slot_j >= a.table.width) continue;
            clash |= a.table.pages[(size_t)sj * a.table.width + slot_j] == page;
        }
        if (__syncthreads_or(clash)) {
            if (tid == 0) atomicCAS(a.error, 0, PAGED_CLASH);
            page = -1;
        }
    }

    float x[8], wv[8], y[8], cs[8], sn[8];
    unpack8(raw, x);
    unpack8(ld16((is_q ? a.qw : a.kw) + d0), wv);
    const int rot = 2 * a.half;
    if (d0 < rot) {
        // half is a multiple of 8, so the 8 dims of a lane share one aligned table pack
        unpack8(ld16(a.cos + (size_t)turn * a.half + d0 % a.half), cs);
        unpack8(ld16(a.sin + (size_t)turn * a.half + d0 % a.half), sn);
    }
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
        if (d0 < rot) y[i] = x[i] * cs[i] + (d0 < a.half ? -partner : partner) * sn[i];
    }
    if (!live) return;
    if (is_q) {
        st16(a.q + ((size_t)r * a.Hq + h) * DH + d0, pack8(y));
        st16(a.gate + ((size_t)r * a.Hq + h) * DH + d0, ld16_stream(src + DH + d0));
    } else if (page >= 0) {
        const size_t at = (((size_t)page * a.table.page_tokens + off) * a.Hk + h) * DH + d0;
        if (is_v)
            st16(a.v_pages + at, raw);
        else
            st16(a.k_pages + at, pack8(y));
    }
}

// ---- attention of one new token per row over its sequence's pages ----
//
// o = sum_t p_t v_t / sum_t p_t, p_t = exp(scale q.k_t - m): one pass with a running maximum and sum.
// Every key and value is read once for all query heads that share it (up to 16 of them, the rows of
// an mma.m16n8k16), which gives at most 16 FLOP per byte: HBM bounds it, not the tensor pipe, and
// tcgen05's 64-row minimum would idle three quarters and more of its rows. So: the copy engine streams
// tiles of 64 tokens through a ring of shared memory that holds most of what an SM has, and four
// warps work on them with plain warp-level MMAs.
//
// The work of a launch is one line of tiles (row by row, key-value head by key-value head, token
// tiles of it) cut into equal runs, one per block, whatever the lengths are. A run's pieces that
// cover a (row, head) whole are finished by the block; the others leave maximum, sum and weighted
// values in float32 in the workspace, and a second kernel joins the parts of each in order.
constexpr int TILE = 64;
constexpr int CONSUMERS = 4, PAGED_THREADS = (CONSUMERS + 1) * 32;
constexpr int MAX_GROUP = 16;   // query heads of one key-value head that a block takes at once
constexpr int MAX_BLOCKS = 296; // two per SM

template <int DH>
struct PCfg {
    static constexpr int BLOCKS_PER_SM = 1;
    static constexpr int HALF_BYTES = TILE * 128;                 // 64 dims of a tile
    static constexpr int KV_BYTES = (DH / 64) * HALF_BYTES;
    static constexpr int STAGE = 2 * KV_BYTES;
    static constexpr int STAGES = DH == 128 ? 6 : 3;
    static constexpr int P_PITCH = TILE + 8;                      // bf16; 144 bytes, so that ldmatrix rows hit all banks
    static constexpr int OFF_P = STAGES * STAGE;
    static constexpr int OFF_F = OFF_P + 16 * P_PITCH * 2;        // float [4][16] maxima, [4][16] sums
    static constexpr int OFF_BAR = OFF_F + 2 * CONSUMERS * 16 * 4;
    static constexpr int SMEM = OFF_BAR + 2 * STAGES * 8 + 64 + 1024;  // and what aligning the base takes
};

struct PagedArgs {
    const bf16 *q, *gate;
    bf16* out;
    const int *seq, *len;
    float* work;
    int* error;
    int rows, Hq, Hk, group, chunk, chunks;  // group = Hq / Hk in `chunks` parts of at most `chunk` heads
    int box;                                 // token rows per copy: a power of two that divides a page
    float scale_log2;
    PageTable table;
};
struct PagedMaps {
    CUtensorMap k, v;
};

// Workspace: [blocks][2] parts of [chunk][DH] weighted values and [chunk] (maximum, sum) pairs, in whole
// 16 bytes, then int4 [blocks] notes.
__host__ __device__ inline size_t part_floats(int chunk, int DH) { return (size_t)chunk * DH + (2 * chunk + 3) / 4 * 4; }

// Tiles of a row over all its heads; 0 for a row that sits out, is empty or is refused.
__device__ __forceinline__ long long row_tiles(const PagedArgs& a, int r, int& tiles) {
    const int n = a.len[r], sq = a.seq ? a.seq[r] : r;
    tiles = 0;
    if (n <= 0 || sq < 0 || sq >= a.table.sequences || n > (long long)a.table.width * a.table.page_tokens) return 0;
    tiles = (n + TILE - 1) / TILE;
    return (long long)tiles * a.Hk * a.chunks;
}

// Position in the line of tiles.
struct Walk {
    int row, head, tile, tiles;  // head: key-value head * chunks + part of its group
    long long left;
};
__device__ __forceinline__ void walk_next_piece(const PagedArgs& a, Walk& w) {
    w.tile = 0;
    if (++w.head < a.Hk * a.chunks) return;
    w.head = 0;
    do {
        w.row++;
    } while (w.row < a.rows && row_tiles(a, w.row, w.tiles) == 0);
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
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

__device__ __forceinline__ float gated(float o, float gate) { return o / (1.f + __expf(-gate)); }

template <int DH>
__global__ void __launch_bounds__(PAGED_THREADS, PCfg<DH>::BLOCKS_PER_SM)
    attn_paged_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ PagedMaps maps) {
    using G = PCfg<DH>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + G::OFF_BAR);
    uint64_t* empty = full + G::STAGES;
    volatile int* gave_up = reinterpret_cast<volatile int*>(empty + G::STAGES);
    __shared__ long long warp_sums[PAGED_THREADS / 32];
    __shared__ Walk begin;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    grid_dep_trigger();
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

    // ---- this block's run of the line of tiles ----
    {
        const int per = (a.rows + PAGED_THREADS - 1) / PAGED_THREADS;
        const int r0 = min(tid * per, a.rows), r1 = min(r0 + per, a.rows);
        long long mine = 0;
        for (int r = r0; r < r1; r++) {
            int tiles;
            mine += row_tiles(a, r, tiles);
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
        // never an empty run between two others: the join follows a piece from block to block
        const long long runs = min((long long)gridDim.x, total), b = blockIdx.x;
        const long long lo = b < runs ? total * b / runs : total, hi = b < runs ? total * (b + 1) / runs : total;
        if (tid == 0 && lo == hi) begin.left = 0;
        if (lo < hi && upto - mine <= lo && lo < upto) {
            long long at = upto - mine;
            for (int r = r0; r < r1; r++) {
                int tiles;
                const long long n = row_tiles(a, r, tiles);
                if (lo < at + n) {
                    const int in_row = (int)(lo - at);  // below 2^31: the host limits a row's tiles
                    begin.row = r;
                    begin.head = in_row / tiles;
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
    // rows without tiles: an empty one has nothing to attend to and gets zeros
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const int n = a.len[r], sq = a.seq ? a.seq[r] : r;
        if (n < 0) continue;
        if (sq < 0 || sq >= a.table.sequences || n > (long long)a.table.width * a.table.page_tokens) {
            if (tid == 0) atomicCAS(a.error, 0, PAGED_BAD_ROW);
        } else if (n == 0) {
            uint32_t* z = reinterpret_cast<uint32_t*>(a.out + (size_t)r * a.Hq * DH);
            for (int i = tid; i < a.Hq * DH / 2; i += PAGED_THREADS) z[i] = 0;
        }
    }
    Walk w = begin;
    auto fail = [&](int code) { atomicCAS(a.error, 0, code); };

    if (warp == CONSUMERS) {
        // ---- copies: the whole warp walks, lane b looks up the page of box b, lane 0 issues ----
        const int boxes = TILE / a.box;
        uint32_t it = 0;
        while (w.left > 0) {
            const int n = a.len[w.row], sq = a.seq ? a.seq[w.row] : w.row;
            const int* pages = a.table.pages + (size_t)sq * a.table.width;
            const int hk = w.head / a.chunks;
            const int end = (int)min((long long)w.tiles, w.tile + w.left);
            for (; w.tile < end; w.tile++, w.left--, it++) {
                const int stage = it % G::STAGES;
                const int t = w.tile * TILE + lane * a.box;
                int at = -1;  // the box's first row in the pools
                if (lane < boxes && t < n) {
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
                if (lane == 0) mbar_expect_tx(&full[stage], (uint32_t)have * a.box * DH * 4);
                __syncwarp();
                if (at >= 0) {
                    unsigned char* dst = smem + stage * G::STAGE + lane * a.box * 128;
#pragma unroll
                    for (int c = 0; c < DH / 64; c++) {
                        tma_load_2d(dst + c * G::HALF_BYTES, &maps.k, hk * DH + c * 64, at, &full[stage]);
                        tma_load_2d(dst + G::KV_BYTES + c * G::HALF_BYTES, &maps.v, hk * DH + c * 64, at, &full[stage]);
                    }
                }
            }
            if (w.left > 0) walk_next_piece(a, w);
        }
    } else {
        constexpr int DW = DH / CONSUMERS, NT = DW / 8;  // dims of the result per warp, in n-tiles of 8
        const uint32_t p_addr = smem_addr(smem + G::OFF_P);
        float* wmax = reinterpret_cast<float*>(smem + G::OFF_F);
        float* wsum = wmax + CONSUMERS * 16;
        const int ra = lane >> 2, rb = ra + 8;  // the two rows (query heads) of this lane's accumulators
        // lane parts of the ldmatrix addresses
        const int k_tok = warp * 16 + (lane >> 4) * 8 + (lane & 7), k_ch = (lane >> 3) & 1;
        const int v_tok = ((lane >> 3) & 1) * 8 + (lane & 7), v_ch = warp * (DW / 8) + (lane >> 4);
        int4 note = make_int4(-1, 0, 0, 0);
        uint32_t it = 0;
        bool ok = true;
        while (w.left > 0) {
            const int n = a.len[w.row];
            const int hk = w.head / a.chunks, part = w.head % a.chunks;
            const int h0 = part * a.chunk, heads = min(a.chunk, a.group - h0);
            const size_t q_row = ((size_t)w.row * a.Hq + (size_t)hk * a.group + h0) * DH;
            uint32_t qf[DH / 16][4];
#pragma unroll
            for (int ks = 0; ks < DH / 16; ks++) {
                const bf16* src = a.q + q_row + ks * 16 + (lane & 3) * 2;
                qf[ks][0] = ra < heads ? *reinterpret_cast<const uint32_t*>(src + (size_t)ra * DH) : 0;
                qf[ks][1] = rb < heads ? *reinterpret_cast<const uint32_t*>(src + (size_t)rb * DH) : 0;
                qf[ks][2] = ra < heads ? *reinterpret_cast<const uint32_t*>(src + (size_t)ra * DH + 8) : 0;
                qf[ks][3] = rb < heads ? *reinterpret_cast<const uint32_t*>(src + (size_t)rb * DH + 8) : 0;
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
                const uint32_t kb = smem_addr(smem + stage * G::STAGE), vb = kb + G::KV_BYTES;
                float s[2][4] = {};
#pragma unroll
                for (int ks = 0; ks < DH / 16; ks++) {
                    const int ch = ks * 2 + k_ch;
                    uint32_t b[4];
                    ldsm4(b, kb + (ch >> 3) * G::HALF_BYTES + k_tok * 128 + (((ch ^ k_tok) & 7) << 4));
                    mma16816(s[0], qf[ks], b[0], b[1]);
                    mma16816(s[1], qf[ks], b[2], b[3]);
                }
                const int left = n - w.tile * TILE;  // valid tokens of the tile, from its first on
                const int c0 = warp * 16 + (lane & 3) * 2;
                float xa = -INFINITY, xb = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const bool in = c0 + j * 8 + e < left;
                        s[j][e] = in ? s[j][e] * a.scale_log2 : -INFINITY;
                        s[j][2 + e] = in ? s[j][2 + e] * a.scale_log2 : -INFINITY;
                        xa = fmaxf(xa, s[j][e]);
                        xb = fmaxf(xb, s[j][2 + e]);
                    }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, o));
                    xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, o));
                }
                if ((lane & 3) == 0) wmax[warp * 16 + ra] = xa, wmax[warp * 16 + rb] = xb;
                consumer_sync();
                float na = ma, nb = mb;
#pragma unroll
                for (int i = 0; i < CONSUMERS; i++) na = fmaxf(na, wmax[i * 16 + ra]), nb = fmaxf(nb, wmax[i * 16 + rb]);
                // a row without a finite score so far keeps offset 0: its terms are exp2(-inf) = 0
                const float oa = na == -INFINITY ? 0.f : na, ob = nb == -INFINITY ? 0.f : nb;
                const float fa = exp2f(ma - oa), fb = exp2f(mb - ob);
                ma = na, mb = nb;
                la *= fa, lb *= fb;
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float p0 = exp2f(s[j][0] - oa), p1 = exp2f(s[j][1] - oa), p2 = exp2f(s[j][2] - ob), p3 = exp2f(s[j][3] - ob);
                    la += p0 + p1, lb += p2 + p3;
                    const uint32_t at = p_addr + (uint32_t)(c0 + j * 8) * 2;
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + ra * G::P_PITCH * 2), "r"(pack2(p0, p1)) : "memory");
                    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at + rb * G::P_PITCH * 2), "r"(pack2(p2, p3)) : "memory");
                }
#pragma unroll
                for (int t = 0; t < NT; t++) acc[t][0] *= fa, acc[t][1] *= fa, acc[t][2] *= fb, acc[t][3] *= fb;
                consumer_sync();
#pragma unroll
                for (int ks = 0; ks < TILE / 16; ks++) {
                    uint32_t pf[4];
                    ldsm4(pf, p_addr + ((lane & 15) * G::P_PITCH + ks * 16 + (lane >> 4) * 8) * 2);
                    const int tok = ks * 16 + v_tok;
                    // values behind the last token may be anything, NaN included: their products with a
                    // probability of zero have to be zero
                    const bool tail = ks * 16 + 16 > left;
#pragma unroll
                    for (int t = 0; t < NT; t += 2) {
                        const int ch = v_ch + t;
                        uint32_t b[4];
                        ldsm4_t(b, vb + (ch >> 3) * G::HALF_BYTES + tok * 128 + (((ch ^ tok) & 7) << 4));
                        if (tail) {
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int t0 = ks * 16 + (e & 1) * 8 + (lane & 3) * 2;
                                b[e] &= (t0 < left ? 0xffffu : 0u) | (t0 + 1 < left ? 0xffff0000u : 0u);
                            }
                        }
                        mma16816(acc[t], pf, b[0], b[1]);
                        mma16816(acc[t + 1], pf, b[2], b[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
            }

            // ---- the piece's end ----
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                la += __shfl_xor_sync(0xffffffffu, la, o);
                lb += __shfl_xor_sync(0xffffffffu, lb, o);
            }
            if ((lane & 3) == 0) wsum[warp * 16 + ra] = la, wsum[warp * 16 + rb] = lb;
            consumer_sync();
            la = lb = 0.f;
#pragma unroll
            for (int i = 0; i < CONSUMERS; i++) la += wsum[i * 16 + ra], lb += wsum[i * 16 + rb];
            const bool whole = from == 0 && end == w.tiles;
            if (whole) {
                const float ia = la == 0.f ? 0.f : 1.f / la, ib = lb == 0.f ? 0.f : 1.f / lb;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const size_t at = q_row + warp * DW + t * 8 + (lane & 3) * 2;
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int row = e ? rb : ra;
                        if (row >= heads) continue;
                        float y0 = acc[t][2 * e] * (e ? ib : ia), y1 = acc[t][2 * e + 1] * (e ? ib : ia);
                        if (a.gate) {
                            const uint32_t g2 = *reinterpret_cast<const uint32_t*>(a.gate + at + (size_t)row * DH);
                            y0 = gated(y0, __uint_as_float(g2 << 16));
                            y1 = gated(y1, __uint_as_float(g2 & 0xffff0000u));
                        }
                        *reinterpret_cast<uint32_t*>(a.out + at + (size_t)row * DH) = pack2(y0, y1);
                    }
                }
            } else {
                // the part that begins a (row, head) lies in place 1, one that continues it in place 0
                const int place = from == 0 ? 1 : 0;
                float* dst = a.work + ((size_t)blockIdx.x * 2 + place) * part_floats(a.chunk, DH);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const int d = warp * DW + t * 8 + (lane & 3) * 2;
                    if (ra < heads) *reinterpret_cast<float2*>(dst + ra * DH + d) = make_float2(acc[t][0], acc[t][1]);
                    if (rb < heads) *reinterpret_cast<float2*>(dst + rb * DH + d) = make_float2(acc[t][2], acc[t][3]);
                }
                float* ml = dst + a.chunk * DH;
                if (warp == 0 && (lane & 3) == 0) {
                    if (ra < heads) ml[2 * ra] = ma, ml[2 * ra + 1] = la;
                    if (rb < heads) ml[2 * rb] = mb, ml[2 * rb + 1] = lb;
                }
                if (place == 1)
                    note.x = w.row, note.y = w.head;
                else
                    note.z = end == w.tiles ? 2 : 1;
            }
            if (w.left > 0) walk_next_piece(a, w);
        }
        if (tid == 0)
            reinterpret_cast<int4*>(a.work + (size_t)gridDim.x * 2 * part_floats(a.chunk, DH))[blockIdx.x] = note;
    }
    // after an abort give copies in flight time to land before the shared memory is released
    if (*gave_up) __nanosleep(1000000);
    __syncthreads();
}

// Joins the parts of the (row, head)s that were cut: block (b, i) takes query head i of the one that
// begins in block b of the first kernel and goes on in the blocks after it, if there is one. The
// order of the sums is fixed by the cut alone.
constexpr int JOIN_WARPS = 8;
template <int DH>
__global__ void __launch_bounds__(JOIN_WARPS * 32) attn_paged_join_kernel(const __grid_constant__ PagedArgs a, int blocks) {
    constexpr int E = DH / 32;
    __shared__ float sums[JOIN_WARPS][DH];
    __shared__ int stop;
    grid_dep_trigger();
    grid_dep_sync();
    const int b = blockIdx.x, i = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t floats = part_floats(a.chunk, DH);
    const int4* notes = reinterpret_cast<const int4*>(a.work + (size_t)blocks * 2 * floats);
    const int4 mine = notes[b];
    if (mine.x < 0) return;
    const int hk = mine.y / a.chunks, h0 = mine.y % a.chunks * a.chunk;
    if (i >= min(a.chunk, a.group - h0)) return;
    if (threadIdx.x == 0) stop = blocks;
    __syncthreads();
    for (int j = b + 1 + threadIdx.x; j < blocks; j += JOIN_WARPS * 32)
        if (notes[j].z != 1) atomicMin(&stop, j);
    __syncthreads();
    const int parts = min(stop, blocks - 1) - b + 1;  // b's place 1, then place 0 of b + 1 .. stop
    auto part = [&](int p) { return a.work + ((size_t)(b + p) * 2 + (p == 0)) * floats; };
    float m = -INFINITY;
    for (int p = lane; p < parts; p += 32) m = fmaxf(m, part(p)[a.chunk * DH + 2 * i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m == -INFINITY) m = 0.f;
    float l = 0.f;
    for (int p = lane; p < parts; p += 32) {
        const float* ml = part(p) + a.chunk * DH + 2 * i;
        l += ml[1] * exp2f(ml[0] - m);
    }
    l = warp_sum(l);
    float acc[E] = {};
    for (int p = warp; p < parts; p += JOIN_WARPS) {
        const float* src = part(p);
        const float f = exp2f(src[a.chunk * DH + 2 * i] - m);
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 x = *reinterpret_cast<const float4*>(src + (size_t)i * DH + e * 32 + lane * 4);
            acc[e] += f * x.x, acc[e + 1] += f * x.y, acc[e + 2] += f * x.z, acc[e + 3] += f * x.w;
        }
    }
#pragma unroll
    for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(&sums[warp][e * 32 + lane * 4]) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= DH) return;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < JOIN_WARPS; w++) y += sums[w][d];
    y = l == 0.f ? 0.f : y / l;
    const size_t at = ((size_t)mine.x * a.Hq + (size_t)hk * a.group + h0 + i) * DH + d;
    if (a.gate) y = gated(y, f32(a.gate[at]));
    a.out[at] = to_bf16(y);
}

// The attention family's error word on the current device, looked up once per device.
int error_word(int** p, int* device) {
    static int* address[64] = {};
    const cudaError_t e = cudaGetDevice(device);
    if (e != cudaSuccess) return e;
    if (*device >= 64) return cudaErrorInvalidDevice;
    if (!address[*device]) {
        int* a = nullptr;
        const int rc = attn_error_address(&a);
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

template <int DH>
int run_paged(const PagedArgs& a, const PagedMaps& maps, int dev, int blocks, cudaStream_t st) {
    using G = PCfg<DH>;
    static bool configured[64] = {};
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(attn_paged_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM);
        if (e != cudaSuccess) return e;
        configured[dev] = true;
    }
    cudaError_t e = launch_dep_family(DEP_ATTENTION, attn_paged_kernel<DH>, blocks, PAGED_THREADS, G::SMEM, st, a, maps);
    if (e != cudaSuccess) return e;
    // always a programmatic dependent: it waits for the first kernel before it reads anything
    e = launch_maybe_dep(true, attn_paged_join_kernel<DH>, dim3(blocks, a.chunk), JOIN_WARPS * 32, 0, st, a, blocks);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace
}  // namespace s1

using namespace s1;

extern "C" int s1_attn_prep_paged(const void* qg, const void* kr, const void* vr, int ld, const void* qw, const void* kw,
                                  const void* cos, const void* sin, int angles, const int* angle, void* q, void* gate,
                                  void* k_pages, void* v_pages, int n_pages, int page_tokens, const int* table,
                                  int table_pages, int n_seqs, const int* seq, const int* pos, int rows, int Hq, int Hk,
                                  int Dh, int half, float eps, void* stream) {
    if ((Dh != 128 && Dh != 256) || Hq <= 0 || Hk <= 0 || Hq > (1 << 20) || Hk > (1 << 20) || rows < 0 || angles < 0 || ld % 8 != 0 ||
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
    const int units = PREP_THREADS / (Dh / 8);
    const dim3 grid(rows, (Hq + 2 * Hk + units - 1) / units);
    if (grid.y > 65535) return cudaErrorInvalidValue;
    int dev = 0;
    const int rc = error_word(&a.error, &dev);
    if (rc != 0) return rc;
    const cudaError_t e = launch_dep(Dh == 256 ? attn_prep_paged_kernel<256> : attn_prep_paged_kernel<128>, grid, PREP_THREADS, 0,
                                     as_stream(stream), a);
    return e != cudaSuccess ? e : cudaGetLastError();
}

extern "C" size_t s1_attention_paged_workspace_floats(int Hq, int Hk, int Dh) {
    if (Hq <= 0 || Hk <= 0 || Hq % Hk != 0 || (Dh != 128 && Dh != 256)) return 0;
    return (size_t)MAX_BLOCKS * (2 * part_floats(std::min(Hq / Hk, MAX_GROUP), Dh) + 4);
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
    if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(q) & 3) ||
        (reinterpret_cast<uintptr_t>(out) & 3) || (reinterpret_cast<uintptr_t>(gate) & 3))
        return cudaErrorInvalidValue;
    if (workspace_floats < s1_attention_paged_workspace_floats(Hq, Hk, Dh)) return cudaErrorInvalidValue;
    PagedArgs a{};
    a.group = Hq / Hk;
    a.chunks = (a.group + MAX_GROUP - 1) / MAX_GROUP;
    a.chunk = (a.group + a.chunks - 1) / a.chunks;
    const long long row_most = ((long long)table_pages * page_tokens + TILE - 1) / TILE * Hk * a.chunks;
    if (row_most > 0x7fffffffLL) return cudaErrorInvalidValue;
    a.q = static_cast<const bf16*>(q), a.gate = static_cast<const bf16*>(gate), a.out = static_cast<bf16*>(out);
    a.seq = seq, a.len = len, a.work = workspace, a.rows = rows, a.Hq = Hq, a.Hk = Hk, a.table = t;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.box = page_tokens % 64 == 0 ? 64 : page_tokens % 32 == 0 ? 32 : 16;
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
    if (!tensor_map_2d(k_pages, pool_rows, width, width, a.box, &maps.k) ||
        !tensor_map_2d(v_pages, pool_rows, width, width, a.box, &maps.v))
        return CS1_ERR_TENSOR_MAP;
    const int per_sm = Dh == 256 ? PCfg<256>::BLOCKS_PER_SM : PCfg<128>::BLOCKS_PER_SM;
    const int blocks = (int)std::min<long long>(std::min(MAX_BLOCKS, sm_count[dev] * per_sm), rows * row_most);
    return Dh == 256 ? run_paged<256>(a, maps, dev, blocks, as_stream(stream)) : run_paged<128>(a, maps, dev, blocks, as_stream(stream));
}
