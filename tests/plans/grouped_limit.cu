// Host-side check of the cut of a grouped product after calls of other sizes.  The runtime calls that the launcher makes are replaced by the ones below,
// which keep a kernel's shared-memory limit as the runtime does: it is what was set last, and no cluster fits that is asked about with more.
// Prints the cut of the last of two calls, in `order` 1 behind a smaller one and otherwise by itself, and with `fail` once behind a question that failed.
#include <cstdio>
#include <cstdlib>
#include <cuda.h>
#include <cuda_runtime.h>
#include <map>

static constexpr int SMS = 148, MAX_SMEM = 232448;
static std::map<const void*, int> limits;
static int fail = 0, wrong = 0, grid = 0, cluster = 1, smem = 0;

static cudaError_t get_device(int* dev) { *dev = 0; return cudaSuccess; }
static cudaError_t device_attribute(int* v, cudaDeviceAttr, int) { *v = SMS; return cudaSuccess; }
static cudaError_t last_error() { return cudaSuccess; }
template <typename K>
static cudaError_t set_attribute(K kernel, cudaFuncAttribute, int value) { limits[(const void*)kernel] = value; return cudaSuccess; }
template <typename K>
static cudaError_t clusters(int* n, K kernel, const cudaLaunchConfig_t* lc) {
  if (fail > 0) { --fail; return cudaErrorUnknown; }
  if ((int)lc->dynamicSmemBytes > limits[(const void*)kernel]) { *n = 0; return cudaSuccess; }
  const unsigned parts = lc->attrs[0].val.clusterDim.x;
  *n = parts == 2 ? 74 : parts == 4 ? 36 : 16;
  return cudaSuccess;
}
template <typename K, typename... Args>
static cudaError_t launch(const cudaLaunchConfig_t* lc, K kernel, Args&&...) {
  if ((int)lc->dynamicSmemBytes > limits[(const void*)kernel]) ++wrong;
  grid = (int)lc->gridDim.x;
  smem = (int)lc->dynamicSmemBytes;
  cluster = lc->numAttrs > 1 ? (int)lc->attrs[1].val.clusterDim.x : 1;
  return cudaSuccess;
}
static CUresult encode(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                       CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill) { return CUDA_SUCCESS; }
static cudaError_t entry_point(const char*, void** fn, unsigned long long, cudaDriverEntryPointQueryResult* found) {
  *fn = reinterpret_cast<void*>(encode);
  *found = cudaDriverEntryPointSuccess;
  return cudaSuccess;
}

#define cudaGetDevice get_device
#define cudaDeviceGetAttribute device_attribute
#define cudaGetLastError last_error
#define cudaFuncSetAttribute set_attribute
#define cudaOccupancyMaxActiveClusters clusters
#define cudaLaunchKernelEx launch
#define cudaGetDriverEntryPoint entry_point
#include "../../fgms_b200/csrc/grouped_umma.cuh"

static void call(int rows, int c_in, int c_out) {
  fgms::GroupedParams p = {};
  p.n_rows = rows; p.c_in = c_in; p.c_out = c_out; p.groups = 1;
  p.a_pitch = c_in;
  p.b_pitch = p.d_pitch = c_out;
  if (fgms::launch_grouped_umma<fgms::GROUPED_FWD>(p, true, nullptr, SMS, MAX_SMEM) != 0) ++wrong;
}

int main(int argc, char** argv) {
  const int order = std::atoi(argv[1]);
  fail = std::atoi(argv[2]);
  if (order == 1) call(1, 768, 768);
  if (order == 2) call(1, 4096, 1024);  // where the question fails, the parts are not shared by this call
  if (order == 1 && cluster < 2) ++wrong;  // the smaller call was to be one of several parts
  call(1, 4096, 1024);
  std::printf("grid %d, clusters of %d, %d bytes, %d wrong\n", grid, cluster, smem, wrong);
  return wrong;
}
