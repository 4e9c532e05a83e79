// Positions and the cache (verinf_amd/csrc/positions.hip) on the CPU, launches and all.
#include "simt_generation.hpp"
#include "positions.hip"
extern "C" const char *simt_error() { return vi::err_buf(); }
