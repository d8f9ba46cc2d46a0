// A CUDA runtime without a GPU, for tests of the library's host code: device memory is host memory, kernels are counted
// and not run, and the n-th allocation from now can be made to fail. Linked with some of the library's objects.
#include <cuda_runtime_api.h>

#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

struct pai_ctx;
void pai_io_destroy(pai_ctx*) {}
void pai_dp_destroy(pai_ctx*) {}

namespace {
struct Block {
  void* p;
  size_t bytes;
};
std::vector<Block> blocks;
long until_failure = -1, launches = 0;
std::string log_text;
cudaError_t make_stream(cudaStream_t* s) {
  *s = reinterpret_cast<cudaStream_t>(malloc(1));
  return cudaSuccess;
}
}  // namespace

extern "C" {
// the test's side
void fake_fail_after(long n) { until_failure = n; }
long fake_blocks() { return (long)blocks.size(); }
long fake_launches() { return launches; }
void* fake_block(size_t bytes) {  // the newest of this size
  for (size_t i = blocks.size(); i-- > 0;)
    if (blocks[i].bytes == bytes) return blocks[i].p;
  return nullptr;
}
const char* fake_log() { return log_text.c_str(); }
void fake_log_clear() { log_text.clear(); }

// the library's side
cudaError_t cudaGetDeviceCount(int* n) { *n = 1; return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetDeviceProperties_v2(cudaDeviceProp* p, int) {
  memset(p, 0, sizeof *p);
  strcpy(p->name, "fake");
  p->major = 10;
  p->multiProcessorCount = 148;
  return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t bytes) {
  if (until_failure == 0) return cudaErrorMemoryAllocation;
  if (until_failure > 0) until_failure--;
  *p = malloc(bytes);
  memset(*p, 0x5a, bytes);
  blocks.push_back({*p, bytes});
  return cudaSuccess;
}
cudaError_t cudaFree(void* p) {
  for (size_t i = 0; i < blocks.size(); i++)
    if (blocks[i].p == p) {
      free(p);
      blocks.erase(blocks.begin() + (long)i);
      break;
    }
  return cudaSuccess;
}
cudaError_t cudaHostAlloc(void** p, size_t bytes, unsigned) { *p = malloc(bytes); return cudaSuccess; }
cudaError_t cudaFreeHost(void* p) { free(p); return cudaSuccess; }
cudaError_t cudaMemset(void* p, int v, size_t n) { log_text += "memset "; memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemsetAsync(void* p, int v, size_t n, cudaStream_t) { memset(p, v, n); return cudaSuccess; }
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) { memmove(d, s, n); return cudaSuccess; }
cudaError_t cudaStreamCreateWithFlags(cudaStream_t* s, unsigned) { return make_stream(s); }
cudaError_t cudaStreamDestroy(cudaStream_t s) { free(s); return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { log_text += "device_synchronize "; return cudaSuccess; }
cudaError_t cudaEventCreate(cudaEvent_t* e) { *e = nullptr; return cudaSuccess; }
cudaError_t cudaEventCreateWithFlags(cudaEvent_t* e, unsigned) { *e = nullptr; return cudaSuccess; }
cudaError_t cudaEventDestroy(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventRecord(cudaEvent_t, cudaStream_t) { return cudaSuccess; }
cudaError_t cudaEventSynchronize(cudaEvent_t) { return cudaSuccess; }
cudaError_t cudaEventElapsedTime(float* ms, cudaEvent_t, cudaEvent_t) { *ms = 0; return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
const char* cudaGetErrorName(cudaError_t) { return "fake"; }
const char* cudaGetErrorString(cudaError_t) { return "fake"; }
cudaError_t cudaFuncSetAttribute(const void*, cudaFuncAttribute, int) { return cudaSuccess; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { launches++; return cudaSuccess; }
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t*, const void*, void**) { launches++; return cudaSuccess; }
cudaError_t cudaStreamBeginCapture(cudaStream_t, cudaStreamCaptureMode) { return cudaSuccess; }
cudaError_t cudaStreamEndCapture(cudaStream_t, cudaGraph_t* g) { *g = nullptr; return cudaSuccess; }
cudaError_t cudaGraphInstantiate(cudaGraphExec_t* e, cudaGraph_t, unsigned long long) { *e = nullptr; return cudaSuccess; }
cudaError_t cudaGraphDestroy(cudaGraph_t) { return cudaSuccess; }
cudaError_t cudaGraphExecDestroy(cudaGraphExec_t) { return cudaSuccess; }
cudaError_t cudaGraphLaunch(cudaGraphExec_t, cudaStream_t) { return cudaSuccess; }
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void*) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
void** __cudaRegisterFatBinary(void*) { static void* handle; return &handle; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, dim3*, dim3*, int*) {}
void __cudaRegisterVar(void**, char*, char*, const char*, int, size_t, int, int) {}
}
