// Verification of drafted tokens against the target's probabilities.
#pragma once

#include "sb_common.cuh"
#include "wait_errors.cuh"

namespace sb {

constexpr int VERIFY_MAX_NODES = 1024;

struct VerifyArgs {
    const float *logits = nullptr;  // row (b, node) at (b*N + node) * ld, n_vocab wide
    const float *draft = nullptr;   // the same layout (ld_draft), or null
    long long ld = 0, ld_draft = 0;
    const int *tokens = nullptr;    // [B][N]
    const int *parents = nullptr;   // [N] (parents_ld 0) or [B][N]
    int parents_ld = 0;
    const float *u = nullptr;       // [B][N]
    const float *noise = nullptr;   // row b at b * ld_noise
    long long ld_noise = 0;
    int B = 0, N = 0, V = 0;
    float temperature = 1.0f;
    int *path = nullptr;      // [B][N], -1 behind the accepted nodes
    int *n_accept = nullptr;  // [B]
    int *next = nullptr;      // [B]
    unsigned *errors = nullptr;  // wait_errors.cuh
};
// Whether every node's row is read before the walk; `part` then holds
// B * N * verify_chunks pairs, else it is null.
bool verify_all_rows(const VerifyArgs &a);
int verify_chunks(const VerifyArgs &a);
int verify_launch(const VerifyArgs &a, float2 *part, cudaStream_t st);

}  // namespace sb
