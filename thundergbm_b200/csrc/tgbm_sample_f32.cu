#include "tgbm_sample_long.cuh"

template bool tgbm::sample_long<float>(const tgbm::SampleArgs &, cudaStream_t);
