// Compilation unit of liblcpp_b200.so: operators over sequences (gated linear recurrence, beam search).
#include "recurrence.cu"
#include "beam.cu"
