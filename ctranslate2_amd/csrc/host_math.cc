#include "host_math.h"

#include <dlfcn.h>

#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <filesystem>
#include <mutex>
#include <stdexcept>
#include <string>
#include <vector>

namespace ct2x {

namespace {

// MKL's single dynamic library (LP64 interface: MKL_INT = int).
using VmlFn = void (*)(int n, const float* a, float* r);

struct Vml {
  VmlFn vs_sin = nullptr;
  VmlFn vs_cos = nullptr;
};

// libmkl_rt loads the rest of MKL when it is first called, and ends the process where that is missing: it is
// used only if core, threading layer and vector functions lie beside it.
bool complete(const void* symbol) {
  Dl_info info;
  if (dladdr(symbol, &info) == 0 || info.dli_fname == nullptr) return false;
  std::error_code error;
  const std::filesystem::path file = std::filesystem::canonical(info.dli_fname, error);
  if (error) return false;
  bool core = false, threads = false, vml = false;
  for (const auto& entry : std::filesystem::directory_iterator(file.parent_path(), error)) {
    const std::string name = entry.path().filename().string();
    core = core || name.rfind("libmkl_core.so", 0) == 0;
    threads = threads || name.rfind("libmkl_intel_thread.so", 0) == 0;
    vml = vml || name.rfind("libmkl_vml_", 0) == 0;
  }
  return core && threads && vml;
}

Vml& vml() {
  static Vml v;
  static std::once_flag once;
  std::call_once(once, [] {
    const char* mode = std::getenv("CT2X_HOST_MATH");
    const std::string want = mode ? mode : "auto";
    if (want == "libm") return;
    std::vector<std::string> dirs = {""};  // "" = the loader's own search path
    for (const char* env : {"CT2X_MKL_PATH", "MKLROOT", "CONDA_PREFIX"}) {
      if (const char* d = std::getenv(env)) {
        dirs.push_back(std::string(d) + "/");
        dirs.push_back(std::string(d) + "/lib/");
        dirs.push_back(std::string(d) + "/lib/intel64/");
      }
    }
    dirs.push_back("/opt/conda/lib/");
    dirs.push_back("/opt/intel/oneapi/mkl/latest/lib/");
    dirs.push_back("/opt/intel/oneapi/mkl/latest/lib/intel64/");
    for (const auto& d : dirs)
      for (const char* name : {"libmkl_rt.so.2", "libmkl_rt.so.1", "libmkl_rt.so"}) {
        void* h = v.vs_sin ? nullptr : dlopen((d + name).c_str(), RTLD_LAZY | RTLD_LOCAL);
        if (!h) continue;
        // (no MKL_Set_Threading_Layer here: the library may be shared with the host application -
        // numpy's, say - and the threading layer is process wide)
        void *sin = dlsym(h, "vsSin"), *cos = dlsym(h, "vsCos");
        if (sin && cos && complete(sin)) {
          v.vs_sin = reinterpret_cast<VmlFn>(sin);
          v.vs_cos = reinterpret_cast<VmlFn>(cos);
        } else {
          (void)dlclose(h);
        }
      }
    if (want == "mkl" && !v.vs_sin)
      throw std::runtime_error("CT2X_HOST_MATH=mkl but no MKL runtime (libmkl_rt.so) was found; set "
                               "CT2X_MKL_PATH");
  });
  return v;
}

void run(VmlFn fn, float (*fallback)(float), int64_t n, const float* x, float* y) {
  if (fn) {
    constexpr int64_t kChunk = 1 << 20;
    for (int64_t i = 0; i < n; i += kChunk)
      fn(static_cast<int>(n - i < kChunk ? n - i : kChunk), x + i, y + i);
    return;
  }
  for (int64_t i = 0; i < n; ++i) y[i] = fallback(x[i]);
}

}  // namespace

void host_vsin(int64_t n, const float* x, float* y) { run(vml().vs_sin, sinf, n, x, y); }
void host_vcos(int64_t n, const float* x, float* y) { run(vml().vs_cos, cosf, n, x, y); }
const char* host_math_backend() { return vml().vs_sin ? "mkl-vml" : "libm"; }

}  // namespace ct2x
