// host.cuh -- host-side plumbing shared by the library's translation units
// (defined in ravel_b200.cu): launch accounting, launch attributes, per-entry
// timing, the device error word, and TMA tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/ravel_b200.h"

namespace ravel {

// SMs of the current device.
int sm_count();

// Called once after every kernel launch of this library: counts it and returns
// RAVEL_OK or RAVEL_ERR_CUDA.
int check_launch();

// Let a kernel be launched with `bytes` of dynamic shared memory beside its static shared memory (the limit is raised
// once per kernel and device where the two pass 48 KB).
int raise_smem(const void* kernel, size_t bytes);

template <typename K>
int set_smem(K kernel, size_t bytes) {
    return raise_smem(reinterpret_cast<const void*>(kernel), bytes);
}

// Launch a kernel that calls grid_wait() (programmatic dependent launch: its blocks may be set up while the
// previous kernel of the stream drains), in clusters of `cluster` blocks where that is more than 1.
template <typename... P, typename... A>
int launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2] = {};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    const int rc = check_launch();
    return e == cudaSuccess ? rc : RAVEL_ERR_CUDA;
}

// Device addresses of the current device's error word and wait limit, for
// kernels of other translation units (looked up once per device).
struct DeviceWords {
    unsigned int* error;
    const unsigned int* wait_limit;
};
int device_words(DeviceWords* out);

// cuTensorMapEncodeTiled of a row-major 2-D tensor (inner x outer elements,
// `pitch` bytes between rows), boxes of box_inner x box_outer, 128-byte swizzle,
// zero fill outside.  type: CU_TENSOR_MAP_DATA_TYPE_*.
int encode_map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, int64_t inner, int64_t outer,
                  int64_t pitch, int box_inner, int box_outer);

// One timing record around the rest of the enclosing entry point (a pair of CUDA
// events while ravel_timing_start's recording is on, nothing otherwise).
class EntryTimer {
  public:
    EntryTimer(const char* entry, void* stream);
    ~EntryTimer();
    EntryTimer(const EntryTimer&) = delete;
    EntryTimer& operator=(const EntryTimer&) = delete;

  private:
    cudaStream_t st_;
    int64_t slot_ = -1;
};
#define RAVEL_TIMED(entry, stream) ravel::EntryTimer ravel_entry_timer_(entry, stream)

}  // namespace ravel
