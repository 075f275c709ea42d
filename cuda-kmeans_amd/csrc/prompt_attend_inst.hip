/* One instantiation of the attention over prompts: KMX_J groups of 32 channels per head (given on the command line). */
#include "prompt_attend_impl.h"

#ifndef KMX_J
#error "compile with -DKMX_J=<groups of 32 channels per head>"
#endif

namespace kmx {

template int launch_prompt_attend<KMX_J>(const PromptAttend& a, bool bf16, const PromptPlan& plan);

} // namespace kmx
