// Attention over the paged cache in 4 bits: many rows a request.
#include "paged_attention_many.h"

namespace shmt {

template void launch_attention_many<4, SHMT_SEEN_CAUSAL>(const AttnArgs &, int, int, unsigned, const AttnScratch &, hipStream_t);

}  // namespace shmt
