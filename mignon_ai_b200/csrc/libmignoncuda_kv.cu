// The translation unit of libmignoncuda.so for the quantised key/value cache and window attention.
#include "mc_kv.cu"
#include "mc_window.cu"
