// attend_wide.h for float16 (a file for each type: they are compiled side by side)
#include "attend_wide.h"

int launch_attend_wide_f16(const AttendArgs& a, const Cut& cut, hipStream_t st) { return launch_wide_of<ODMKV_F16>(a, cut, st); }
