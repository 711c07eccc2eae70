// Attention with queries of type f16.
#include "attend_launch.h"

template int launch_attend_few<2, 4>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_many<2, 4>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_step<2>(const AttendArgs &, const SelectArgs &, hipStream_t);
