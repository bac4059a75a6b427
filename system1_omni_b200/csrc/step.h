// What the decode operators share: the table of sequences that own rows of a step and the slots
// that hold what a sequence carries from one step to the next, checked on the device.
#pragma once
#include "common.cuh"

namespace s1 {

// Sequence i owns rows [start[i], start[i+1]) (start null: row i), begins with what slot_in[i] of a
// pool holds (negative: zeros) and leaves its result in slot_out[i] (negative: it sits this step out).
struct StepSeqs {
    const int *start, *slot_in, *slot_out;
    int nseq, rows, n_slots;
};

// Codes that the delta-rule step operators leave in their device error word.
enum { STEP_BAD_ROWS = 60, STEP_BAD_SLOT = 61, STEP_SLOT_CLASH = 62 };

struct StepSeq {
    int row0, rows, in, out;  // rows < 0: nothing to do
    int code;                 // why it is refused, 0: it is not
};

__device__ __forceinline__ StepSeq step_sequence(const StepSeqs& s, int i) {
    StepSeq q;
    q.code = 0;
    q.in = s.slot_in[i];
    q.out = s.slot_out[i];
    q.row0 = s.start ? s.start[i] : i;
    q.rows = (s.start ? s.start[i + 1] : i + 1) - q.row0;
    if (q.out < 0)
        q.rows = -1;
    else if (q.row0 < 0 || q.rows < 0 || q.row0 > s.rows - q.rows)
        q.code = STEP_BAD_ROWS, q.rows = -1;
    else if (q.in >= s.n_slots || q.out >= s.n_slots)
        q.code = STEP_BAD_SLOT, q.rows = -1;
    return q;
}

// Whether one of the sequences `first`, `first + stride`, ... writes what sequence i reads or
// writes, or reads what it writes. Such sequences would race, so every one of them is refused.
__device__ __forceinline__ bool step_clash(const StepSeqs& s, int i, int in, int out, int first, int stride) {
    bool clash = false;
    for (int j = first; j < s.nseq; j += stride) {
        const int jo = s.slot_out[j], ji = s.slot_in[j];
        clash |= j != i && jo >= 0 && (jo == out || ji == out || jo == in);
    }
    return clash;
}

// The same for `n` sequences of a block, i0 and on, at once: every other sequence's slots are looked up among theirs,
// which for many sequences takes a fraction of comparing all with all in every block. What they write and what they
// begin with are looked up apart: sequences may share a slot to begin with, and all of a block that do are one chain, in which
// only slots that someone writes are looked up; a bit of another hash keeps those off it that merely fall into its place.
// A chain of slots to write is short, or its sequences are refused. All threads of the block call it.
constexpr int STEP_ROWS = 128;
struct StepLookup {
    static constexpr int HASH = 512;
    struct Slots {
        int first[HASH], next[STEP_ROWS], slot[STEP_ROWS];  // chains of 1 + entry
        uint32_t bits[HASH];                                // of the slots in a chain
        __device__ __forceinline__ void put(int e, int s) {
            slot[e] = s;
            if (s < 0) return;
            next[e] = atomicExch(&first[hash(s)], e + 1);
            atomicOr(&bits[hash(s)], bit(s));
        }
    } outs, ins;
    bool clashes[STEP_ROWS];
    static __device__ __forceinline__ uint32_t hash(int s) { return (uint32_t)s * 2654435769u >> 23; }
    static __device__ __forceinline__ uint32_t bit(int s) { return 1u << ((uint32_t)s * 2654435769u >> 18 & 31); }
    // Marks the block's sequences that have slot s in `of`, but for `own`, the one that it is looked up for.
    __device__ __forceinline__ void mark(const Slots& of, int s, int own) {
        if (!(of.bits[hash(s)] & bit(s))) return;
        for (int e = of.first[hash(s)]; e > 0; e = of.next[e - 1])
            if (of.slot[e - 1] == s && e - 1 != own) clashes[e - 1] = true;
    }
    template <int THREADS>
    __device__ __forceinline__ void find(const StepSeqs& s, int i0, int n) {
        const int tid = threadIdx.x;
        for (int e = tid; e < HASH; e += THREADS) outs.first[e] = ins.first[e] = 0, outs.bits[e] = ins.bits[e] = 0;
        __syncthreads();
        for (int e = tid; e < n; e += THREADS) {
            clashes[e] = false;
            outs.put(e, s.slot_out[i0 + e]);
            ins.put(e, s.slot_in[i0 + e]);
        }
        __syncthreads();
        constexpr int AT_ONCE = 4;
        for (int j0 = tid; j0 < s.nseq; j0 += AT_ONCE * THREADS) {
            int out[AT_ONCE], in[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                const int j = min(j0 + u * THREADS, s.nseq - 1);
                out[u] = s.slot_out[j], in[u] = s.slot_in[j];
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) {
                const int own = min(j0 + u * THREADS, s.nseq - 1) - i0;
                if (out[u] < 0) continue;
                mark(outs, out[u], own);
                mark(ins, out[u], own);
                if (in[u] >= 0) mark(outs, in[u], own);
            }
        }
        __syncthreads();
    }
};

// (At most 65535 sequences: a grid dimension.)
inline bool step_seqs_ok(const StepSeqs& s) {
    return s.nseq >= 0 && s.nseq <= 65535 && s.rows >= 0 && s.n_slots >= 0 && (s.nseq == 0 || (s.slot_in && s.slot_out));
}

}  // namespace s1
