// Compilation unit of liblcpp_b200.so: softmax cross entropy over a vocabulary, from hidden states.
#include "cross_entropy.cu"
