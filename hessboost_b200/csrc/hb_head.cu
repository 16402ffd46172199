// What the embedding-head operators share on the host (hb_head.h).
#include "hb_head.h"

#include <atomic>

namespace hb {
namespace head {
namespace {
thread_local std::string g_head_error;
std::atomic<int> g_sms[64];
}  // namespace

hb_status fail(hb_status st, const std::string& what) {
  g_head_error = what;
  return st;
}

void begin_call() {
  if (!g_head_error.empty()) g_head_error.clear();
}

int sm_count(int device) {
  const bool kept = device >= 0 && device < 64;
  int n = kept ? g_sms[device].load(std::memory_order_relaxed) : 0;
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) {
      cudaGetLastError();
      return 1;  // no such device: the call is refused later
    }
    if (kept) g_sms[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

hb_status launched(const char* where) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return HB_OK;
  return fail(HB_DEVICE_FAILED, std::string(where) + ": " + cudaGetErrorString(e));
}

}  // namespace head
}  // namespace hb

extern "C" const char* hb_head_last_error(void) { return hb::head::g_head_error.c_str(); }
