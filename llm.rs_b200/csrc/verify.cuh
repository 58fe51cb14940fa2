// verify.cuh - verification of drafted tokens (host interface).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace llmrs {

struct VerifyParams {
    const void *logits;       // [n_rows][ld]
    long long ld;
    int dtype, vocab, n_rows, n_seqs;
    int n_drafts;             // entries of draft, rows of q
    const int *row_start;     // [n_seqs + 1]
    const int *draft;         // [n_drafts], packed: one fewer than the rows of each sequence
    const float *q;           // [n_drafts][ldq] the drafting model's probabilities; nullptr: each draft was certain
    long long ldq;
    const float *u;           // [n_rows] uniform draws
    const float *temperature; // [n_seqs] or nullptr (1)
    int *tokens;              // [n_rows]
    int *accepted;            // [n_seqs]
    float *probs;             // [n_rows] or nullptr
    uint32_t *err;
};

// tokens are counted in 32 bits, in steps that reach some thousands past the last one
constexpr int VERIFY_MAX_VOCAB = 1 << 30;

size_t verify_workspace(int n_rows, int vocab);
// set kernel attributes on the current device (once per context, outside capture)
int verify_prepare(void);
int verify_launch(const VerifyParams &p, void *ws, cudaStream_t stream);

} // namespace llmrs
