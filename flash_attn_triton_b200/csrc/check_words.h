// The words in mapped host memory that value checks are answered in (decode.cu): a call takes one, gives it to a kernel that
// writes the result with kCheckDone set, waits for that and gives it back.
#pragma once
#include <cstdint>

#include <cuda_runtime.h>

namespace fa {

// Index of a word, its address on `device` (the current one) at *dptr; -1 (error set) without one.
int take_check_word(bool ticket, int device, uint32_t** dptr);
// Waits until the kernel that was given the word has written it.
int await_check_word(int i, uint32_t* failed, cudaStream_t st);
// queued: a kernel that writes the word is on a stream.
void give_check_word(int i, bool queued);

}  // namespace fa
