// How a cut row's pieces leave their denominators to the merge (the block-scaled cache's kernels), in a file of its own so
// that it also compiles for the host.
#pragma once
#include <stdbool.h>

#include "page_run.h"   // KVQ_HOST_DEVICE

// The sign bit marks the last piece, a zero's too, and nothing is added to the number: the largest weight of a denominator
// is 2^-32 (BLOCK_REF). Slot 0 of a row that was not cut is marked as well (-1); a cut row has two pieces or more. (The static
// cache's kernels store -2 - l: there l is about 1 or more; 2^-32 would be lost.)
KVQ_HOST_DEVICE float last_piece_sum(float l) { return -l; }
KVQ_HOST_DEVICE bool is_last_piece(float stored) { return __builtin_signbit(stored); }
KVQ_HOST_DEVICE float piece_sum(float stored) { return __builtin_fabsf(stored); }
