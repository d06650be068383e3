#include "tgbm_sample_long.cuh"

template bool tgbm::sample_long<__nv_bfloat16>(const tgbm::SampleArgs &, cudaStream_t);
