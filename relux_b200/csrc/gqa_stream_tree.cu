// Tree steps over the bf16 cache.
#include "gqa_stream_kernel.cuh"

namespace relux {

int32_t launch_gqa_stream_tree(Pool* p, const GqaStreamCommon& c, const GqaSeq* seqs, const int8_t* parents, int workers) {
  return launch_variant<kTree>(p, c, seqs, parents, workers);
}

}  // namespace relux
