// Attention of a few rows: queries of type f32.
#include "attend_few.h"

template int launch_attend_few<3>(const AttendArgs &, int64_t, hipStream_t);
