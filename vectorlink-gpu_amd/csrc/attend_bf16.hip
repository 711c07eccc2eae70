// Attention of a few rows: queries of type bf16.
#include "attend_few.h"

template int launch_attend_few<1>(const AttendArgs &, int64_t, hipStream_t);
