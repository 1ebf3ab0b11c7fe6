// Compilation unit of liblcpp_b200.so: gated delta rule.
#include "delta_rule.cu"
