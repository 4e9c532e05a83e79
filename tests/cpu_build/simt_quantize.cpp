// Rows to 8-bit integers (verinf_amd/csrc/quantize.hip) on the CPU, launches and all.
#include "simt_inference.hpp"
#include "quantize.hip"
extern "C" const char *simt_error() { return vi::err_buf(); }
