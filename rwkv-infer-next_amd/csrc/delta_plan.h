// delta_plan.h -- where the chunks of the gated delta rule's rows lie in its workspace.  Host arithmetic on sizes alone, and what the
// kernels compute of it.
#pragma once
#include <stdint.h>

#include <algorithm>

#ifdef __HIPCC__
#define DELTA_BOTH __host__ __device__ inline
#else
#define DELTA_BOTH inline
#endif

namespace delta {

constexpr int kChunk = 64;

// A slot holds a chunk.  Rows of T tokens have theirs one after another.  Of ragged rows the host knows the number and the tokens of all;
// those of at most token_len tokens have no chunks.  Row n, whose first token is the one of number `first`, begins at slot
//     first / 64 + n, room enough whatever the rows, or
//     first / 2^shift, 2^shift <= 32 and <= token_len + 1: a longer row of L tokens has ceil(L / 64) chunks, L / 2^shift is no less, and
//     neither is the distance to the slot where the next one begins;
// whichever needs fewer in all: few long rows the first, many short ones, of which few can be long, the second (1024 single tokens 65
// slots, not 1040).
struct Slots {
    int32_t shift, rows;  // rows: 1 where each row moves those behind it on by a slot
    int64_t count;
};
inline Slots ragged_slots(int64_t num_seqs, int64_t total_tokens, int32_t token_len) {
    int32_t shift = 0;
    while (shift < 5 && (2 << shift) <= token_len + 1) ++shift;
    const Slots apart{6, 1, total_tokens / kChunk + num_seqs}, close{shift, 0, (total_tokens >> shift) + 1};
    return close.count < apart.count ? close : apart;
}
inline Slots row_slots(int64_t num_seqs, int32_t T) { return {0, 0, num_seqs * (((int64_t)T + kChunk - 1) / kChunk)}; }
DELTA_BOTH int64_t ragged_slot(int32_t shift, int32_t rows, int32_t n, int64_t first) { return (first >> shift) + (rows ? n : 0); }

// How many ragged rows can be longer than token_len.
inline int64_t long_rows(int64_t num_seqs, int64_t total_tokens, int32_t token_len) {
    return std::min(num_seqs, total_tokens / ((int64_t)token_len + 1));
}

}  // namespace delta
