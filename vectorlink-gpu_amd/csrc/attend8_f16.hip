// Attention over a cache in 8 bits with queries of type f16.
#include "attend_launch.h"
#include "weigh.h"

template int launch_attend_few<2, 8>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_many<2, 8>(const AttendArgs &, int64_t, hipStream_t);
template int launch_weigh_rows<2>(const AttendArgs &, hipStream_t);
