// Attention with queries of type f32.
#include "attend_launch.h"

template int launch_attend_few<3>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_many<3>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_step<3>(const AttendArgs &, const SelectArgs &, hipStream_t);
