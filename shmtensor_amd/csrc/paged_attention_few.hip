// Attention over the paged cache in 4 bits: few rows a request.
#include "paged_attention_few.h"

namespace shmt {

template void launch_attention_few<4, SHMT_SEEN_CAUSAL>(const AttnArgs &, int, int, int, unsigned, const AttnScratch &,
                                                    hipStream_t);

}  // namespace shmt
