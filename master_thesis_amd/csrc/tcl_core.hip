// Error reporting and version of libtcl_hip.so.
#include "tcl_common.h"
#include <map>
#include <mutex>
#include <utility>

namespace tcl {

static thread_local char g_err[512] = "";

int set_error(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int check_launch(const char *what) {
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(TCL_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
  return TCL_OK;
}

// Dynamic LDS above 64 KB needs the kernel's attribute raised (per device; asked again only for more than was granted).
bool lds_ready(const void *kernel, size_t lds) try {
  if (lds <= 64 * 1024) return true;
  static std::mutex mu;
  static std::map<std::pair<const void *, int>, size_t> granted;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  std::lock_guard<std::mutex> lock(mu);
  size_t &have = granted[std::make_pair(kernel, dev)];
  if (lds > have) {
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) {
      (void)hipGetLastError();   // a refusal is not an error of a later call
      return false;
    }
    have = lds;
  }
  return true;
} catch (...) {   // no exception leaves through the C entry points
  return false;
}

}  // namespace tcl

extern "C" int tcl_version(void) { return TCL_VERSION; }
extern "C" const char *tcl_last_error(void) { return tcl::g_err; }
