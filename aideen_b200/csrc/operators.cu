// Errors and device facts shared by the operators on caller-owned tensors.
#include "operators.cuh"

namespace aideen {
namespace {
thread_local const char *g_why = "";
constexpr int kMaxDevices = 64;
int g_sms[kMaxDevices] = {};

int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : -1;
}
}  // namespace

void op_set_error(const char *why) { g_why = why ? why : ""; }

// One value per device, which every thread computes alike.
int op_sm_count() {
  const int dev = current_device();
  if (dev < 0) return 148;
  if (!g_sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    g_sms[dev] = n;
  }
  return g_sms[dev];
}

}  // namespace aideen

extern "C" const char *aideen_operator_error(void) { return aideen::g_why; }

extern "C" int aideen_operator_check(void *stream) {
  using namespace aideen;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaStreamSynchronize(st);
  unsigned int v = 0;
  if (e == cudaSuccess) e = linear_ce_timeout(&v);
  if (e != cudaSuccess) return op_cuda(e);
  if (v) {
    op_set_error("a bounded wait ran out (outputs since the last check are invalid)");
    return AIDEEN_E_TIMEOUT;
  }
  return AIDEEN_OK;
}
