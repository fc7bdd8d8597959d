// Verification of drafted tokens (k_verify.hip).
#pragma once
#include <cstddef>
#include <cstdint>

#include "sq_common.h"

namespace sq {

constexpr int kVerifySeqs = 256;       // sequences of one launch: their counts travel as kernel arguments
constexpr size_t kVerifyDrafts = 1024;  // drafts of one sequence at most

struct VerifyBatch {
    uint32_t target0[kVerifySeqs];  // first target row of a sequence; sequence s's first draft row is target0[s] - s
    uint16_t n[kVerifySeqs];
    uint32_t n_seqs;
};
struct VerifyArgs {
    const float* target;
    size_t target_stride;
    const float* draft;  // null: a draft is its token with probability 1
    size_t draft_stride;
    const uint32_t* tokens;
    const float* u;
    int vocab;
    double inv_t;  // log2(e) / temperature; 0: greedy
};
struct VerifyResult {
    uint32_t accepted, token, bad, pad;
};

// Whether one launch takes so many target and draft rows.
bool verify_fits(size_t rows, int vocab);
// Bytes of workspace for `rows` target and draft rows and n_seqs sequences.
size_t verify_ws_bytes(size_t rows, size_t n_seqs, int vocab);
int launch_verify(hipStream_t s, const VerifyBatch& b, const VerifyArgs& a, size_t target_rows, size_t draft_rows,
                  void* ws, VerifyResult* results);

}  // namespace sq
