// ABI version and the thread-local error channel of the C ABI.
#include <mutex>
#include <vector>

#include "common.h"

namespace ff {

static thread_local std::string g_error;

void set_error(const std::string& msg) { g_error = msg; }
void clear_error() { g_error.clear(); }

int fail(int code, const std::string& msg) {
  g_error = msg;
  return code;
}

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(FF_ELAUNCH, std::string(what) + ": " + hipGetErrorString(e));
  return FF_OK;
}

int64_t resident_blocks(const void* kernel, int block, size_t smem) {
  struct Entry {
    const void* kernel;
    int device, block;
    size_t smem;
    int64_t blocks;
  };
  static std::mutex mu;
  static std::vector<Entry> cache;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  {
    std::lock_guard<std::mutex> lock(mu);
    for (const Entry& e : cache)
      if (e.kernel == kernel && e.device == dev && e.block == block && e.smem == smem) return e.blocks;
  }
  int per_cu = 0, cus = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, block, smem) != hipSuccess ||
      hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || per_cu <= 0 || cus <= 0) {
    (void)hipGetLastError();
    return 0;
  }
  const int64_t blocks = static_cast<int64_t>(per_cu) * cus;
  std::lock_guard<std::mutex> lock(mu);
  cache.push_back({kernel, dev, block, smem, blocks});
  return blocks;
}

static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }  // b > 0

bool apart(const Extent& a, const Extent& b) {
  if (a.len <= 0 || b.len <= 0) return true;
  int64_t common[2];  // the pitch of a dimension, -1 where the two differ
  int64_t inner_a[2], inner_b[2], ext_a = a.len, ext_b = b.len;
  for (int d = 0; d < 2; ++d) {
    common[d] = a.n[d] <= 1 ? (b.n[d] <= 1 ? 0 : b.pitch[d]) : (b.n[d] <= 1 || a.pitch[d] == b.pitch[d] ? a.pitch[d] : -1);
    inner_a[1 - d] = a.len + (a.n[d] > 1 ? (a.n[d] - 1) * a.pitch[d] : 0);  // extent over one step of the other dimension
    inner_b[1 - d] = b.len + (b.n[d] > 1 ? (b.n[d] - 1) * b.pitch[d] : 0);
    ext_a += inner_a[1 - d] - a.len;
    ext_b += inner_b[1 - d] - b.len;
  }
  if (a.at < b.at ? b.at - a.at >= static_cast<uint64_t>(ext_a) : a.at - b.at >= static_cast<uint64_t>(ext_b)) return true;
  const int64_t off = static_cast<int64_t>(b.at - a.at);
  for (int d = 0; d < 2; ++d)
    if (common[d] > 0) {
      const int64_t r = off - floor_div(off, common[d]) * common[d];
      if (inner_a[d] <= r && inner_b[d] <= common[d] - r) return true;
    }
  if (common[0] < 0 || common[1] < 0) return false;
  // Runs i0, i1 steps from each other start off + i0 pitch0 + i1 pitch1 apart; they meet if that lies in (-len b, len a).
  for (int64_t i1 = -(a.n[1] - 1); i1 <= b.n[1] - 1; ++i1) {
    const int64_t x = off + i1 * common[1];
    if (common[0] == 0) {
      if (-b.len < x && x < a.len) return false;
      continue;
    }
    const int64_t lo = floor_div(-b.len - x, common[0]) + 1, hi = -floor_div(x - a.len, common[0]) - 1;
    if (lo <= hi && lo <= b.n[0] - 1 && hi >= -(a.n[0] - 1)) return false;
  }
  return true;
}

}  // namespace ff

extern "C" int ff_abi_version(void) { return 4; }

extern "C" const char* ff_last_error(void) { return ff::g_error.c_str(); }
