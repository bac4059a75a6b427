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

// Codes that the step operators leave in a family's device error word.
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

// (At most 65535 sequences: a grid dimension, and every sequence is compared with every other.)
inline bool step_seqs_ok(const StepSeqs& s) {
    return s.nseq >= 0 && s.nseq <= 65535 && s.rows >= 0 && s.n_slots >= 0 && (s.nseq == 0 || (s.slot_in && s.slot_out));
}

}  // namespace s1
