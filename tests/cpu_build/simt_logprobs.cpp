// Log probabilities (verinf_amd/csrc/logprobs.hip) on the CPU, launches and all.
#include "simt_inference.hpp"
#include "logprobs.hip"
extern "C" const char *simt_error() { return vi::err_buf(); }
extern "C" long simt_groups_met() { return simt::groups_met; }
