// seq_kernels.h -- launchers of the sequence operators (layer norm, causal
// convolution, selective scan), internal to libsdtw_b200.  The argument blocks
// are the public ones of include/sdtw_b200.h.
#pragma once

#include <cuda_runtime.h>

#include "../../include/sdtw_b200.h"

namespace sdtw {

// layer_norm.cu
cudaError_t launch_layer_norm_fwd(const sdtw_layer_norm_args& a, cudaStream_t st);
cudaError_t launch_layer_norm_bwd(const sdtw_layer_norm_args& a, cudaStream_t st);
size_t layer_norm_bwd_ws(long long rows, int dim);

// causal_conv.cu
constexpr int kConvMaxWidth = 8;
cudaError_t launch_conv_fwd(const sdtw_conv_args& a, cudaStream_t st);
cudaError_t launch_conv_bwd(const sdtw_conv_args& a, cudaStream_t st);
cudaError_t launch_conv_step(const sdtw_conv_args& a, cudaStream_t st);
size_t conv_bwd_ws(int batch, int length, int dim, int width);

// selective_scan_fwd.cu, selective_scan_bwd.cu
constexpr int kScanMaxState = 64;
// Lanes over the states of a feature (4 states each).
constexpr int scan_lanes(int nstate) {
    int nl = 1;
    while (4 * nl < nstate) nl *= 2;
    return nl;
}
// Time steps between two states that the forward stores for the backward.
constexpr int kScanSave = 16;
struct ScanSplit {
    int nseg, seglen;
};
ScanSplit scan_split(int batch, int length, int dim, int groups, int nstate);
cudaError_t launch_scan_fwd(const sdtw_scan_args& a, cudaStream_t st);
cudaError_t launch_scan_bwd(const sdtw_scan_args& a, cudaStream_t st);
cudaError_t launch_scan_step(const sdtw_scan_args& a, cudaStream_t st);
size_t scan_states(int batch, int length, int dim, int nstate);
size_t scan_fwd_ws(int batch, int length, int dim, int groups, int nstate);
size_t scan_bwd_ws(int batch, int length, int dim, int groups, int nstate);

}  // namespace sdtw
