// Attention of trees over the paged cache in 8 bits.
#include "paged_attention_few.h"
#include "paged_attention_many.h"

namespace shmt {

template void launch_attention_few<8, SHMT_SEEN_TREE>(const AttnArgs &, int, int, int, unsigned, const AttnScratch &,
                                                    hipStream_t);
template void launch_attention_many<8, SHMT_SEEN_TREE>(const AttnArgs &, int, int, unsigned, const AttnScratch &, hipStream_t);

}  // namespace shmt
