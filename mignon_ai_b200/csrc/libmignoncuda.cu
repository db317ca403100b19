// The engine's translation unit of libmignoncuda.so: its kernels and C-ABI are compiled together so
// device globals (the error word) and shared device helpers need no separate device linking. The
// key/value cache and window attention, which share no device state with it, are
// libmignoncuda_kv.cu; the two compile side by side.
#include "mc_host.cu"
#include "mc_gemm.cu"
#include "mc_modelfile.cu"
#include "mc_block.cu"
#include "mc_block_decode.cu"
#include "mc_attn.cu"
#include "mc_head.cu"
#include "mc_policy.cu"
#include "mc_tiny.cu"
#include "mc_engine_host.cu"
#include "mc_api.cu"
#include "mc_sched.cu"
#include "mc_convert.cu"
#include "mc_selftest.cu"
#include "mc_probe.cu"
