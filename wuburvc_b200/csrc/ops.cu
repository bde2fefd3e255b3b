// ops.cu — the transformer training operators' device status word.
//
// Their calls are asynchronous, so a bounded wait that expires inside a kernel cannot be reported by
// the call that launched it: the kernel records it in one word per device, which wubu_b200_ops_sync
// reads and clears.
#include <mutex>

#include "ops.cuh"

namespace wb {

static __device__ int g_ops_status;

int* ops_status_word() {
  constexpr int kMaxDevices = 64;
  static std::mutex mu;
  static int* at[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
  // a thread that has made no CUDA call yet (an autograd worker) has no current context, which the
  // driver's tensor-map encoding needs
  static thread_local bool in_context = false;
  if (!in_context && cudaSetDevice(dev) != cudaSuccess) return nullptr;
  in_context = true;
  std::lock_guard<std::mutex> lk(mu);
  if (!at[dev]) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_ops_status) != cudaSuccess) return nullptr;
    at[dev] = static_cast<int*>(p);
  }
  return at[dev];
}

int ops_sms() {
  static std::atomic<int> sms[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  n = sms[dev].load();
  if (!n && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) sms[dev].store(n);
  return n;
}

}  // namespace wb

extern "C" int wubu_b200_ops_sync(void* stream) {
  cudaStream_t st = (cudaStream_t)stream;
  int* word = wb::ops_status_word();
  int code = 0;
  cudaError_t e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && word) e = cudaMemcpyAsync(&code, word, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess && word) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && code) e = cudaMemsetAsync(word, 0, sizeof(int), st);
  if (e != cudaSuccess || !word) {
    fprintf(stderr, "wuburvc_b200: CUDA error %s\n", cudaGetErrorString(e));
    return WUBU_B200_ERR_CUDA;
  }
  if (code) fprintf(stderr, "wuburvc_b200: kernel reported error %d\n", code);
  return code ? WUBU_B200_ERR_TIMEOUT : WUBU_B200_OK;
}
