// Instantiation unit of the decode kernels for head dim 128 and f16 queries over 8-bit
// rows with a scale for each token and kv head: the split partial kernel (both tile scans)
// and the per-sequence kernel.
#include "split_kernels.h"

namespace mxfa {

int launch_rows_128_f16(const DecodeParams &p, const Grid &g, int kind, bool wave_scan,
                       hipStream_t st) {
  return launch_rows_hd<128, F16>(p, g, kind, wave_scan, st);
}

int launch_seq_rows_128_f16(const DecodeParams &p, int kind, hipStream_t st) {
  return launch_seq_rows_hd<128, F16>(p, kind, st);
}

}  // namespace mxfa
