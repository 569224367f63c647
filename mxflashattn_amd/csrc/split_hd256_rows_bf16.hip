// Instantiation unit of the decode kernels for head dim 256 and bf16 queries over 8-bit
// rows with a scale for each token and kv head: the split partial kernel (both tile scans)
// and the per-sequence kernel.
#include "split_kernels.h"

namespace mxfa {

int launch_rows_256_bf16(const DecodeParams &p, const Grid &g, int kind, bool wave_scan,
                       hipStream_t st) {
  return launch_rows_hd<256, BF16>(p, g, kind, wave_scan, st);
}

int launch_seq_rows_256_bf16(const DecodeParams &p, int kind, hipStream_t st) {
  return launch_seq_rows_hd<256, BF16>(p, kind, st);
}

}  // namespace mxfa
