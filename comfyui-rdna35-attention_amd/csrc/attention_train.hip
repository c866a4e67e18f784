// The forward of a training step: the dense attention kernels with grouped key
// heads, a key count per batch entry and the rows' log sums as an output
// (attention.hip compiled with PISA_ATTENTION_TRAIN), built with the
// max-memory-clause machine scheduler like the other dense kernels (build_lib.py).
#define PISA_ATTENTION_TRAIN 1
#include "attention.hip"
