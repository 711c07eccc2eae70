// Attention over a cache in 8 bits with queries of type bf16.
#include "attend_launch.h"
#include "weigh.h"

template int launch_attend_few<1, 8>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_many<1, 8>(const AttendArgs &, int64_t, hipStream_t);
template int launch_weigh_rows<1>(const AttendArgs &, hipStream_t);
