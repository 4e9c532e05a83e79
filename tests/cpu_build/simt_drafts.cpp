// Drafts (verinf_amd/csrc/drafts.hip) on the CPU, launches and all.
#include "simt_generation.hpp"
#include "drafts.hip"
extern "C" const char *simt_error() { return vi::err_buf(); }
