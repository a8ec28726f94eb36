// Words in which the kernels of the speculative decoding operators record that
// a bounded wait gave up.  They lie in pinned host memory that every device
// reads and writes in place, so the host looks at them without a copy.
#pragma once

namespace sb {

enum WaitError { WAIT_TREE_ROWS, WAIT_TREE_TC, WAIT_TREE_F32, WAIT_VERIFY, WAIT_ERRORS };

// The first recorded error, which is cleared, or -1.
inline int take_wait_error(volatile unsigned *words) {
    for (int i = 0; i < WAIT_ERRORS; i++)
        if (words[i]) {
            words[i] = 0;
            return i;
        }
    return -1;
}

#ifdef __CUDACC__
// The words (WAIT_ERRORS of them, allocated by the first call; also during a capture).
int wait_error_words(unsigned **words);
// Reports (and clears) a recorded error; SB_OK before the words exist.
int wait_error_check();
__device__ __forceinline__ void wait_failed(unsigned *words, WaitError e) { *static_cast<volatile unsigned *>(words + e) = 1u; }
#endif

}  // namespace sb
