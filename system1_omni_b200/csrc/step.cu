// The Gated DeltaNet operators of the tokens after a prefill: the convolution and the gates of new
// rows behind kept ones, and the gated delta rule token by token.
//
// Float32 from the inputs to one rounding at the end. The prefill's operators round in between where
// the model stores a tensor (the convolution before its SiLU), so a step's bf16 results differ from
// theirs by a step of bf16 at times; what a slot keeps is the same.
#include <algorithm>
#include <type_traits>

#include "cs1_ops.h"
#include "s1_executor.h"
#include "status.h"
#include "step.h"

namespace s1 {
namespace {

constexpr int D = 128;  // key and value dim of the delta rule

// ---- delta rule ----
// Per token, with k = k/|k|, q = scale q/|q| (both with 1e-6 under the root) and the state S [key, value]:
//   d = beta (v - e^g k^T S),  S <- e^g S + k d^T,  o = q^T S = e^g q^T S_before + (q.k) d.
// The value columns are independent of one another, so a warp takes CW of them with all 128 keys and
// keeps its part of S in registers over the window's tokens: S is read once and written once, and
// both products of a token come from one pass over the registers. Lane l owns columns
// 4 (l % (CW/4)) .. + 3 of the keys l / (CW/4), + RG, ...; the sums over keys are closed by shuffles. The warps
// of a (sequence, head) are one block and prepare the rows (norms, gates) of up to CHUNK tokens together.
typedef unsigned long long f32x2;  // two floats, the unit of the packed FMA
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 two(float lo, float hi) {
    f32x2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void lds(uint32_t at, f32x2& a, f32x2& b) { asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(at)); }
// Volatile: the update reads the keys again rather than hold 64 registers of them from the products on.
__device__ __forceinline__ f32x2 lds_again(uint32_t at) {
    f32x2 a;
    asm volatile("ld.volatile.shared.b64 %0, [%1];" : "=l"(a) : "r"(at));
    return a;
}
__device__ __forceinline__ void split(f32x2 x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ void unpack4(uint2 p, float (&x)[4]) {
    x[0] = __uint_as_float(p.x << 16), x[1] = __uint_as_float(p.x & 0xffff0000u);
    x[2] = __uint_as_float(p.y << 16), x[3] = __uint_as_float(p.y & 0xffff0000u);
}

// HBM bounds it with one token a sequence: 64 KiB of state in, 64 KiB out per head, all of a block's reads
// issued at once. Measured at 193 sequences of 48 heads (1.22 GB): 186 us, 6.55 TB/s; columns per warp and
// blocks per SM at least: 32 and 2: 189 us, 16 and 2: 228, 8 and 2: 276 (narrower warps fetch pieces of lines).
// Windows are bound by latency (shared memory first, then the FMAs), with the 2.7 warps per scheduler that such
// registers leave: 37 windows of 1 to 9 tokens, 32 heads, 38 us (the bytes alone 13), the FMA pipe active for 33 %.
// The products of eight tokens at once on the tensor cores with the state split into three bf16 took 39 to 43
// us, two resident blocks that prefetch the next state into shared memory 49 to 55, twice the warps with half the
// columns 44 to 52, the longest windows first 37.5, and a state kept divided by its decay, a quarter fewer FMAs, 37.5
// too, with 10.2 for 9.6 us for 3 windows of 9 tokens.
constexpr int CW = 32, CHUNK = 8, FEW_HEADS = 296, MANY_SEQS = 2560;

__device__ __forceinline__ void copy16(const void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int WARPS, bool MANY>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 4 ? 3 : 8)
    gdn_step_kernel(const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v,
                    const float* __restrict__ g, const bf16* __restrict__ beta, bf16* __restrict__ o, int H, int group,
                    float scale, float* states, size_t slot_stride, const StepSeqs seqs, int per, int* error) {
    constexpr int CL = CW / 4, RG = 32 / CL, RL = D / RG;  // lanes over columns, groups of lanes over keys, keys per lane
    constexpr int SPLIT = D / CW / WARPS;  // blocks of a (sequence, head)
    __shared__ __align__(16) float4 kkqq[CHUNK][D];  // k, k, q, q
    __shared__ __align__(16) bf16 ks[CHUNK][D], qs[CHUNK][D], vs[CHUNK][D];
    __shared__ float4 gates[CHUNK];                  // e^g, beta, q.k
    grid_dep_trigger();
    grid_dep_sync();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = (int)(blockIdx.x / SPLIT % H), i0 = (int)(blockIdx.x / SPLIT / H) * (MANY ? per : 1);
    __shared__ typename std::conditional<MANY, StepLookup, int>::type lookup;
    if constexpr (MANY) lookup.template find<WARPS * 32>(seqs, i0, min(per, seqs.nseq - i0));
    int i = i0;
    do {
        if (MANY && i > i0) __syncthreads();  // the rows of the one before have been read
        const StepSeq sq = step_sequence(seqs, i);
        if (sq.code && threadIdx.x == 0) atomicCAS(error, 0, sq.code);
        if (sq.rows < 0) continue;
        const int c0 = ((int)(blockIdx.x % SPLIT) * WARPS + warp) * CW + lane % CL * 4, r0 = lane / CL;
        const int hk = h / group, HK = H / group;

        // Rows t0 .. of a chunk as they are. The first ones are asked for before the state, which they would queue behind.
        float g_mine = 0.f, beta_mine = 0.f;  // of row t0 + threadIdx.x
        auto fetch = [&](int t0) {
            const int nt = min(CHUNK, sq.rows - t0);
            for (int e = threadIdx.x; e < nt * (D / 8); e += WARPS * 32) {
                const int t = e / (D / 8), d = e % (D / 8) * 8;
                const size_t row = (size_t)sq.row0 + t0 + t;
                copy16(&ks[t][d], k + (row * HK + hk) * D + d);
                copy16(&qs[t][d], q + (row * HK + hk) * D + d);
                copy16(&vs[t][d], v + (row * H + h) * D + d);
            }
            if ((int)threadIdx.x < nt) {
                const size_t at = ((size_t)sq.row0 + t0 + threadIdx.x) * H + h;
                g_mine = g[at], beta_mine = f32(beta[at]);
            }
        };
        fetch(0);

        ulonglong2 S[RL];
        if (sq.in >= 0) {
            const float* src = states + (size_t)sq.in * slot_stride + ((size_t)h * D + r0) * D + c0;
#pragma unroll
            for (int j = 0; j < RL; j++) S[j] = *reinterpret_cast<const ulonglong2*>(src + (size_t)j * RG * D);
        } else {
#pragma unroll
            for (int j = 0; j < RL; j++) S[j] = make_ulonglong2(0, 0);
        }
        bool clash;
        if constexpr (MANY)
            clash = lookup.clashes[i - i0];
        else
            clash = step_clash(seqs, i, sq.in, sq.out, threadIdx.x, WARPS * 32);
        copies_wait();
        if (__syncthreads_or(clash)) {
            if (threadIdx.x == 0) atomicCAS(error, 0, STEP_SLOT_CLASH);
            continue;
        }

#pragma unroll 1
        for (int t0 = 0; t0 < sq.rows; t0 += CHUNK) {
            const int nt = min(CHUNK, sq.rows - t0);
            if (t0 > 0) {
                __syncthreads();  // the rows before have been read
                fetch(t0);
                copies_wait();
                __syncthreads();
            }
#pragma unroll 1
            for (int t = warp; t < nt; t += WARPS) {
                float kv[4], qv[4];
                unpack4(*reinterpret_cast<const uint2*>(&ks[t][lane * 4]), kv);
                unpack4(*reinterpret_cast<const uint2*>(&qs[t][lane * 4]), qv);
                float kk = 0.f, qq = 0.f, qk = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) kk += kv[e] * kv[e], qq += qv[e] * qv[e], qk += kv[e] * qv[e];
                kk = rsqrtf(warp_sum(kk) + 1e-6f);
                qq = rsqrtf(warp_sum(qq) + 1e-6f) * scale;
                qk = warp_sum(qk) * kk * qq;
#pragma unroll
                for (int e = 0; e < 4; e++) kkqq[t][lane * 4 + e] = make_float4(kv[e] * kk, kv[e] * kk, qv[e] * qq, qv[e] * qq);
                if (lane == 0) gates[t].z = qk;
            }
            if ((int)threadIdx.x < nt) gates[threadIdx.x].x = expf(g_mine), gates[threadIdx.x].y = beta_mine;
            __syncthreads();
#pragma unroll 1
            for (int t = 0; t < nt; t++) {
                const uint32_t rows_at = (uint32_t)__cvta_generic_to_shared(&kkqq[t][r0]);
                f32x2 k01 = 0, k23 = 0, q01 = 0, q23 = 0;
#pragma unroll
                for (int j = 0; j < RL; j++) {
                    f32x2 kk, qq;
                    lds(rows_at + j * RG * 16, kk, qq);
                    k01 = fma2(kk, S[j].x, k01);
                    k23 = fma2(kk, S[j].y, k23);
                    q01 = fma2(qq, S[j].x, q01);
                    q23 = fma2(qq, S[j].y, q23);
                }
                float ks[4], qs[4], vv[4], d[4], y[4];
                split(k01, ks[0], ks[1]);
                split(k23, ks[2], ks[3]);
                split(q01, qs[0], qs[1]);
                split(q23, qs[2], qs[3]);
#pragma unroll
                for (int m = CL; m < 32; m <<= 1)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        ks[e] += __shfl_xor_sync(0xffffffffu, ks[e], m);
                        qs[e] += __shfl_xor_sync(0xffffffffu, qs[e], m);
                    }
                const float4 gt = gates[t];
                unpack4(*reinterpret_cast<const uint2*>(&vs[t][c0]), vv);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    d[e] = gt.y * (vv[e] - gt.x * ks[e]);
                    y[e] = gt.x * qs[e] + gt.z * d[e];
                }
                if (r0 == 0) {
                    uint2 p;
                    p.x = pack2(y[0], y[1]);
                    p.y = pack2(y[2], y[3]);
                    *reinterpret_cast<uint2*>(o + (((size_t)sq.row0 + t0 + t) * H + h) * D + c0) = p;
                }
                const f32x2 decay = two(gt.x, gt.x), d01 = two(d[0], d[1]), d23 = two(d[2], d[3]);
#pragma unroll
                for (int j = 0; j < RL; j++) {
                    const f32x2 kk = lds_again(rows_at + j * RG * 16);
                    S[j].x = fma2(decay, S[j].x, mul2(kk, d01));
                    S[j].y = fma2(decay, S[j].y, mul2(kk, d23));
                }
            }
        }
        if (sq.rows == 0 && sq.in == sq.out) continue;
        float* dst = states + (size_t)sq.out * slot_stride + ((size_t)h * D + r0) * D + c0;
#pragma unroll
        for (int j = 0; j < RL; j++) *reinterpret_cast<ulonglong2*>(dst + (size_t)j * RG * D) = S[j];
    } while (MANY && ++i < min(i0 + per, seqs.nseq));
}

// ---- convolution and gates ----
// y_t = silu(sum_j w_j x_{t-3+j}) per channel, the rows before a sequence's first out of its slot's
// tail [3, channels] (x_{-3}, x_{-2}, x_{-1}, before the convolution). A thread walks the window's rows
// for 8 channels with the three rows before in registers; the last row of blocks computes the gates.
//
// Bound by the latency of its three trips (slots, rows, results) and by issue slots, some 400 instructions a
// warp. Measured at 193 sequences of 10240 channels (32 MB, 4.8 us of HBM): 8.1 us; 2, 3 and 4 sequences per
// block, which load the weights once, 8.1, 9.3 and 8.0. One sequence: 2.2 us.
constexpr int CONV_THREADS = 128, CONV_MANY = 4096;

template <bool MANY>
__global__ void __launch_bounds__(CONV_THREADS)
    gdn_conv_gates_step_kernel(const bf16* __restrict__ qkv, int ld, const bf16* __restrict__ w, bf16* __restrict__ q,
                               bf16* __restrict__ k, bf16* __restrict__ v, int key_dim, int value_dim, int conv_blocks,
                               const bf16* __restrict__ b, const bf16* __restrict__ a, const bf16* __restrict__ A_log,
                               const bf16* __restrict__ dt_bias, bf16* __restrict__ beta, float* __restrict__ g, int H,
                               bf16* tails, size_t slot_stride, const StepSeqs seqs, int per, int* error) {
    __shared__ bool clashes[CONV_THREADS / 32];
    __shared__ typename std::conditional<MANY, StepLookup, int>::type lookup;
    grid_dep_trigger();
    grid_dep_sync();
    const int channels = 2 * key_dim + value_dim;
    const int c0 = ((int)blockIdx.x * CONV_THREADS + (int)threadIdx.x) * 8;
    const bool conv = (int)blockIdx.x < conv_blocks && c0 < channels;
    // weights, kept rows and the first new row are all asked for before anything waits
    uint4 wraw[4] = {}, x[4] = {};
    if (conv) {
#pragma unroll
        for (int j = 0; j < 4; j++) wraw[j] = ld16(w + (size_t)c0 * 4 + j * 8);
    }
    const int i0 = blockIdx.y * (MANY ? per : 1);
    if constexpr (MANY) lookup.template find<CONV_THREADS>(seqs, i0, min(per, seqs.nseq - i0));
    int i = i0;
    do {
        const StepSeq sq = step_sequence(seqs, i);
        if (sq.code && threadIdx.x == 0) atomicCAS(error, 0, sq.code);
        if (sq.rows < 0) continue;
        if (conv) {
            if (sq.in >= 0) {
                const bf16* src = tails + (size_t)sq.in * slot_stride + c0;
#pragma unroll
                for (int j = 0; j < 3; j++) x[j] = ld16(src + (size_t)j * channels);
            } else if (MANY) {
#pragma unroll
                for (int j = 0; j < 3; j++) x[j] = make_uint4(0, 0, 0, 0);
            }
            if (sq.rows > 0) x[3] = ld16_stream(qkv + (size_t)sq.row0 * ld + c0);
        }
        bool clash;
        if constexpr (MANY) {
            clash = lookup.clashes[i - i0];
        } else {
            clash = __any_sync(0xffffffffu, step_clash(seqs, i, sq.in, sq.out, threadIdx.x, CONV_THREADS));
            if ((threadIdx.x & 31) == 0) clashes[threadIdx.x >> 5] = clash;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < CONV_THREADS / 32; j++) clash |= clashes[j];
        }
        if (clash) {
            if (threadIdx.x == 0) atomicCAS(error, 0, STEP_SLOT_CLASH);
            continue;
        }
        if ((int)blockIdx.x >= conv_blocks) {
            for (int e = threadIdx.x; e < sq.rows * H; e += CONV_THREADS) {
                const size_t row = (size_t)sq.row0 + e / H;
                const int h = e % H;
                beta[row * H + h] = to_bf16(sigmoid(f32(b[row * ld + h])));
                const float z = f32(a[row * ld + h]) + f32(dt_bias[h]);
                g[row * H + h] = -expf(f32(A_log[h])) * (z > 20.f ? z : log1pf(expf(z)));
            }
            continue;
        }
        if (!conv) continue;
        float wf[8][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float tmp[8];
            unpack8(wraw[j], tmp);
#pragma unroll
            for (int e = 0; e < 8; e++) wf[(j * 8 + e) / 4][(j * 8 + e) % 4] = tmp[e];
        }
        bf16* dst;
        int dld, dc;
        if (c0 < key_dim)
            dst = q, dld = key_dim, dc = c0;
        else if (c0 < 2 * key_dim)
            dst = k, dld = key_dim, dc = c0 - key_dim;
        else
            dst = v, dld = value_dim, dc = c0 - 2 * key_dim;
#pragma unroll 1
        for (int t = 0; t < sq.rows; t++) {
            const size_t row = (size_t)sq.row0 + t;
            if (t > 0) x[3] = ld16_stream(qkv + row * ld + c0);
            float x0[8], x1[8], x2[8], x3[8], y[8];
            unpack8(x[0], x0);
            unpack8(x[1], x1);
            unpack8(x[2], x2);
            unpack8(x[3], x3);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float acc = wf[e][0] * x0[e];
                acc = fmaf(wf[e][1], x1[e], acc);
                acc = fmaf(wf[e][2], x2[e], acc);
                acc = fmaf(wf[e][3], x3[e], acc);
                y[e] = silu_fast(acc);
            }
            st16(dst + row * dld + dc, pack8(y));
            x[0] = x[1];
            x[1] = x[2];
            x[2] = x[3];
        }
        bf16* keep = tails + (size_t)sq.out * slot_stride + c0;
#pragma unroll
        for (int j = 0; j < 3; j++) st16(keep + (size_t)j * channels, x[j]);
    } while (MANY && ++i < min(i0 + per, seqs.nseq));
}

// The delta-rule step operators' error word on the current device, looked up once per device.
int error_word(int** p) {
    static int* address[64] = {};
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= 64) return cudaErrorInvalidDevice;
    if (!address[dev]) {
        int* a = nullptr;
        const int rc = step_error_address(STEP_GDN, &a);
        if (rc != 0) return rc;
        address[dev] = a;
    }
    *p = address[dev];
    return 0;
}

}  // namespace
}  // namespace s1

using namespace s1;

extern "C" int s1_gdn_step(const void* q, const void* k, const void* v, const float* g, const void* beta, void* o, int rows,
                           int H, int HK, float scale, float* states, int n_slots, size_t slot_stride, const int* start,
                           const int* slot_in, const int* slot_out, int nseq, void* stream) {
    const StepSeqs seqs{start, slot_in, slot_out, nseq, rows, n_slots};
    if (!step_seqs_ok(seqs) || H <= 0 || HK <= 0 || H % HK != 0 || slot_stride < (size_t)H * D * D || slot_stride % 4 != 0)
        return cudaErrorInvalidValue;
    if (nseq == 0) return cudaSuccess;
    if (!states || !aligned16(states)) return cudaErrorInvalidValue;
    if (rows > 0 && (!q || !k || !v || !g || !beta || !o || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o)))
        return cudaErrorInvalidValue;
    // few heads to step: a block per warp's columns, so that four times as many SMs take part (32 heads: 3.3 us for 4.6; from some 600 heads on it is slower)
    const long long heads = (long long)nseq * H;
    if (heads > 0x7fffffffLL / 4) return cudaErrorInvalidValue;
    const bool few = heads <= FEW_HEADS;
    int* error = nullptr;
    const int rc = error_word(&error);
    if (rc != 0) return rc;
    // Many sequences: several to a block, which looks all others up at once, where every block would compare all with
    // one. 4 heads, one to a block and several: 2048 sequences 183 and 199 us, 4096: 437 and 396, 16384: 3.5 and 1.6 ms.
    const int per = nseq > MANY_SEQS ? (int)std::min<long long>(STEP_ROWS, heads / 4096) : 1;
    const bool many = per > 1;
    const long long blocks = few ? 4 * heads : many ? (long long)((nseq + per - 1) / per) * H : heads;
    const cudaError_t e = launch_dep(few ? gdn_step_kernel<1, false> : many ? gdn_step_kernel<4, true> : gdn_step_kernel<4, false>, (unsigned)blocks,
                                     few ? 32 : 128, 0, as_stream(stream), static_cast<const bf16*>(q), static_cast<const bf16*>(k),
                                     static_cast<const bf16*>(v), g, static_cast<const bf16*>(beta), static_cast<bf16*>(o), H, H / HK,
                                     scale, states, slot_stride, seqs, per, error);
    return e != cudaSuccess ? e : cudaGetLastError();
}

extern "C" int s1_gdn_conv_gates_step(const void* qkv, int ld, const void* w, void* q, void* k, void* v, int rows, int key_dim,
                                      int value_dim, const void* b, const void* a, const void* A_log, const void* dt_bias,
                                      void* beta, float* g, int H, void* tails, int n_slots, size_t slot_stride,
                                      const int* start, const int* slot_in, const int* slot_out, int nseq, void* stream) {
    const StepSeqs seqs{start, slot_in, slot_out, nseq, rows, n_slots};
    if (!step_seqs_ok(seqs) || key_dim <= 0 || value_dim <= 0 || key_dim % 8 != 0 || value_dim % 8 != 0 || H <= 0 || ld % 8 != 0 ||
        (long long)ld < 2LL * key_dim + value_dim || ld < H || 2LL * key_dim + value_dim > 0x7fffffffLL)
        return cudaErrorInvalidValue;
    const int channels = 2 * key_dim + value_dim;
    if (slot_stride < 3 * (size_t)channels || slot_stride % 8 != 0 || (long long)rows * H > 0x7fffffffLL)
        return cudaErrorInvalidValue;
    if (nseq == 0) return cudaSuccess;
    if (!tails || !aligned16(tails) || !w || !aligned16(w) || !A_log || !dt_bias) return cudaErrorInvalidValue;
    if (rows > 0 && (!qkv || !q || !k || !v || !b || !a || !beta || !g || !aligned16(qkv) || !aligned16(q) || !aligned16(k) ||
                     !aligned16(v)))
        return cudaErrorInvalidValue;
    int* error = nullptr;
    const int rc = error_word(&error);
    if (rc != 0) return rc;
    const int conv_blocks = (channels / 8 + CONV_THREADS - 1) / CONV_THREADS;
    // Several sequences to a block as in s1_gdn_step. 10240 channels, one to a block and several: 1500 sequences 55 and 68 us,
    // 4096: 181 and 162; 1536 channels, 16384: 480 and 174 us, 65535: 11.2 and 0.68 ms (the bytes alone 61 and 245), whether
    // they begin in slots of their own or in one. What is left beside the bytes: every block reads all slots, and a thread has one
    // sequence's rows in flight.
    const int per = nseq >= CONV_MANY ? std::min(STEP_ROWS, nseq / 512) : 1;
    const cudaError_t e = launch_dep(
        per > 1 ? gdn_conv_gates_step_kernel<true> : gdn_conv_gates_step_kernel<false>, dim3(conv_blocks + 1, (nseq + per - 1) / per),
        CONV_THREADS, 0, as_stream(stream),
        static_cast<const bf16*>(qkv), ld, static_cast<const bf16*>(w), static_cast<bf16*>(q), static_cast<bf16*>(k),
        static_cast<bf16*>(v), key_dim, value_dim, conv_blocks, static_cast<const bf16*>(b), static_cast<const bf16*>(a),
        static_cast<const bf16*>(A_log), static_cast<const bf16*>(dt_bias), static_cast<bf16*>(beta), g, H,
        static_cast<bf16*>(tails), slot_stride, seqs, per, error);
    return e != cudaSuccess ? e : cudaGetLastError();
}
