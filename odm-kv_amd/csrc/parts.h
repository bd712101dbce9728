// Where partial results of attention over pages lie in its workspace.  By itself, so that the host's tests compile what the entry points do.
#pragma once

#include <stddef.h>

#include "../../include/odmkv.h"

// Of `parts` results, and `common` more of what rows have in common: where what begins, in floats behind the workspace's 16-byte aligned begin, and how many there are.  Results are written 16 bytes
// at a time: each kind begins on as many, however many logarithms lie in front of it.
struct PartPlaces { size_t lse, common_out, common_lse, floats; };
static inline PartPlaces part_places(size_t parts, size_t common) {
    PartPlaces p;
    p.lse = parts * ODMKV_HEAD_DIM;
    p.common_out = (p.lse + parts + 3) & ~(size_t)3;
    p.common_lse = p.common_out + common * ODMKV_HEAD_DIM;
    p.floats = p.common_lse + common;
    return p;
}
