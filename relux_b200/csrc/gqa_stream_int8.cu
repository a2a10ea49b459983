// GQA decode and verify steps over the 8-bit cache.
#include "gqa_stream_kernel.cuh"

namespace relux {

int32_t launch_gqa_stream_int8(Pool* p, const GqaStreamCommon& c, const GqaSeq* seqs, int workers) {
  return launch_variant<kInt8>(p, c, seqs, nullptr, workers);
}

}  // namespace relux
