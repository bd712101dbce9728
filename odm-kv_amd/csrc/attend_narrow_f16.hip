// attend_narrow.h for float16 (a file for each type: they are compiled side by side)
#include "attend_narrow.h"

int launch_attend_narrow_f16(const AttendArgs& a, const Cut& cut, hipStream_t st) { return launch_narrow_of<ODMKV_F16>(a, cut, st); }
