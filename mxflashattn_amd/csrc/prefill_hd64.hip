// Instantiation unit of the paged prefill kernels for head dim 64.
#include "prefill_kernels.h"

namespace mxfa {

int launch_prefill_64(const PrefillParams &p, int items, bool bf16, int cache, hipStream_t st) {
  return launch_prefill_hd<64>(p, items, bf16, cache, st);
}

}  // namespace mxfa
