// What kernels report through the session's host-mapped error words.
#pragma once

#include <string>

#include "../../include/ort_cuda.h"
#include "ptx.cuh"

namespace ortc {

// Kernels write codes into the host-mapped error words: a bounded wait that gave up,
// lengths and pages that do not fit.  Reported once, all of them; the status is the
// wait's when there is one.
inline int take_kernel_errors(volatile int* words, std::string* msg) {
  int rc = ORT_CUDA_OK;
  for (int i = 0; i < kErrorWords; i++) {
    const int code = words[i];
    if (code == 0) continue;
    words[i] = 0;
    if (!msg->empty()) *msg += "; ";
    if (rc == ORT_CUDA_OK) rc = i == 0 ? ORT_CUDA_ERR_TIMEOUT : ORT_CUDA_ERR_INVALID_ARG;
    switch (code) {
      case KERR_PAGED_LENGTH:
        *msg += "paged KV cache: cu_seqlens and past_lens do not fit num_tokens, max_seq, "
                "shared_len or max_pages * page_size; the sequence was left out";
        break;
      case KERR_PAGED_PAGE:
        *msg += "paged KV cache: block_table names a page outside [0, num_pages); its tokens "
                "were left out";
        break;
      case KERR_PAGED_POSITION:
        *msg += "paged KV cache: a position is outside the cos/sin caches; its token was left out";
        break;
      default:
        *msg += "a kernel wait exceeded its bound (code " + std::to_string(code) +
                "); the kernel stopped and returned";
    }
  }
  return rc;
}

}  // namespace ortc
