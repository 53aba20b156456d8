// Error state and version entry points of the C ABI.
#include <stdarg.h>

#include <algorithm>

#include "common.h"

namespace la {

static thread_local char g_last_error[512] = "";

void set_error(const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
}

int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
  return code;
}

int num_cus() {
  static thread_local int cached_dev = -1, cached = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 256;
  if (dev != cached_dev) {
    int v = 0;
    cached = hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0
                 ? v
                 : 256;
    cached_dev = dev;
  }
  return cached;
}

// Two runs share a byte where the distance of their starts is above -a.run and below b.run:
// whether a sum of terms c s, lo <= c <= hi, added to the distance of the bases is.  The
// largest stride first; a term's c is only tried where the rest can still make up for it.
struct OverlapTerm {
  int64_t s, lo, hi;
};
static bool overlap_from(const OverlapTerm *t, int n, int64_t at, int64_t low, int64_t high, int *left) {
  if (n == 0) return at > low && at < high;
  int64_t neg = 0, pos = 0;
  for (int i = 1; i < n; ++i) {
    neg += t[i].lo * t[i].s;
    pos += t[i].hi * t[i].s;
  }
  // (floors of quotients of any sign)
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t c0 = std::max(t->lo, -floor_div(at + pos - low - 1, t->s));
  const int64_t c1 = std::min(t->hi, floor_div(high - 1 - neg - at, t->s));
  for (int64_t c = c0; c <= c1; ++c) {
    if (--*left < 0) return true;
    if (overlap_from(t + 1, n - 1, at + c * t->s, low, high, left)) return true;
  }
  return false;
}

bool overlap_runs(const Cover &a, const Cover &b) {
  OverlapTerm t[8];
  int n = 0;
  for (const Cover *x : {&a, &b})
    for (const Cover::Dim &d : x->dim) {
      if (d.stride == 0) continue;
      int i = 0;
      while (i < n && t[i].s != d.stride) ++i;
      if (i == n) t[n++] = OverlapTerm{d.stride, 0, 0};
      if (x == &a) t[i].hi += d.count - 1;
      else t[i].lo -= d.count - 1;
    }
  std::sort(t, t + n, [](const OverlapTerm &x, const OverlapTerm &y) { return x.s > y.s; });
  int left = 4096;
  return overlap_from(t, n, a.p - b.p, -a.run, b.run, &left);
}

bool overlap_self(const Cover &a) {
  if (a.run == 0) return false;
  Cover::Dim d[4];
  int n = 0;
  for (const Cover::Dim &x : a.dim)
    if (x.count > 1) d[n++] = x;
  std::sort(d, d + n, [](const Cover::Dim &x, const Cover::Dim &y) { return x.stride < y.stride; });
  int64_t extent = a.run;
  for (int i = 0; i < n; ++i) {
    if (d[i].stride < extent) return true;
    extent += d[i].stride * (d[i].count - 1);
  }
  return false;
}

}  // namespace la

extern "C" int la_abi_version(void) { return LA_ABI_VERSION; }

extern "C" const char *la_last_error(void) { return la::g_last_error; }
