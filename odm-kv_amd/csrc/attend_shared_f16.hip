// The fp16 kernels of attend_shared.h, in a file of their own: the compiler takes them beside the others.
#include "attend_shared.h"

int launch_attend_shared_f16(const AttendArgs& a, int workgroups, hipStream_t st) { return launch_shared_of<ODMKV_F16>(a, workgroups, st); }
