// Tree steps over the 8-bit cache.
#include "gqa_stream_kernel.cuh"

namespace relux {

int32_t launch_gqa_stream_tree_int8(Pool* p, const GqaStreamCommon& c, const GqaSeq* seqs, const int8_t* parents, int workers) {
  return launch_variant<kTree + kInt8>(p, c, seqs, parents, workers);
}

}  // namespace relux
