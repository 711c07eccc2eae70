// Attention with queries of type bf16.
#include "attend_launch.h"

template int launch_attend_few<1>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_many<1>(const AttendArgs &, int64_t, hipStream_t);
template int launch_attend_step<1>(const AttendArgs &, const SelectArgs &, hipStream_t);
