/* One instantiation of the attention over the 4-bit cache: KMX_J groups of 32 channels per head (given on the command line). */
#include "cache4_attend_impl.h"

#ifndef KMX_J
#error "compile with -DKMX_J=<groups of 32 channels per head>"
#endif

namespace kmx {

template int launch_attend4<KMX_J>(Attend4 a, const Plan4& plan);

} // namespace kmx
