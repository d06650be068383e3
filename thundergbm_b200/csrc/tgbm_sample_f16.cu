#include "tgbm_sample_long.cuh"

template bool tgbm::sample_long<__half>(const tgbm::SampleArgs &, cudaStream_t);
