// attend_narrow.h for bfloat16 (a file for each type: they are compiled side by side)
#include "attend_narrow.h"

int launch_attend_narrow_bf16(const AttendArgs& a, const Cut& cut, hipStream_t st) { return launch_narrow_of<ODMKV_BF16>(a, cut, st); }
