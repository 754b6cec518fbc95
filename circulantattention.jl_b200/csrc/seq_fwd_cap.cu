// Attention on token sequences, forward: the kernels of one kind of scores.
#include "seq_fwd.cuh"

template int ca::umma_fwd<ca::kCap>(const ca::SeqArgs&, const ca::FwdMaps&, int, bool, dim3, cudaStream_t);
