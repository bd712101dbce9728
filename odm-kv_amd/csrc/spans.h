// Packed rows: where a row's tokens begin and how many they are, by offsets that nobody on the host has seen.  By itself, so that the host can compile what the kernel does.
#pragma once

#include <hip/hip_runtime.h>

struct Span { int begin, n; };

// The tokens from `first` to before `last` of `all` that there are: within those whatever the two say, and none where they do not ascend.  (Both are brought within them before one
// is taken from the other: the difference of what comes in may pass 32 bits.)
__host__ __device__ static inline Span span_of(int first, int last, int all) {
    const int begin = first < 0 ? 0 : first < all ? first : all, end = last < begin ? begin : last < all ? last : all;
    return {begin, end - begin};
}
