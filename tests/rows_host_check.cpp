// The row operators' rules that only the host decides, checked without a device:
// which outputs are stored with the non-temporal hint, and what overlaps. Built
// for the host alone; the addresses are never followed.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "ps_rows.hpp"

#define CHECK(cond)                                              \
  do {                                                           \
    if (!(cond)) {                                               \
      std::printf("line %d: not so: %s\n", __LINE__, #cond);     \
      return 1;                                                  \
    }                                                            \
  } while (0)

namespace {

ps_rows rows(uintptr_t at, long long n, long long cols, long long ld, int dtype) {
  return {reinterpret_cast<void*>(at), n, cols, ld, dtype};
}

// Byte by byte: whether two matrices share one.
bool share(const ps_rows& a, const ps_rows& b) {
  std::vector<char> taken(4096);
  const auto each = [](const ps_rows& m, auto&& f) {
    const size_t size = ps::dtype_size(m.dtype);
    for (long long r = 0; r < m.rows; ++r)
      for (size_t c = 0; c < size_t(m.cols) * size; ++c)
        f(reinterpret_cast<uintptr_t>(m.data) + size_t(r * m.ld) * size + c);
  };
  each(a, [&](uintptr_t p) { taken[p] = 1; });
  bool shared = false;
  each(b, [&](uintptr_t p) { shared = shared || taken[p]; });
  return shared;
}

int overlaps() {
  std::srand(3);
  int met = 0, apart = 0;
  for (int i = 0; i < 200000; ++i) {
    const long long ld = 1 + std::rand() % 12;
    const auto some = [&](long long pitch) {
      const long long n = std::rand() % 5, cols = 1 + std::rand() % pitch;
      return rows(4 * (1 + std::rand() % 60), n, cols, n == 1 ? cols : pitch, PS_F32);
    };
    const ps_rows a = some(ld), b = some(ld), flat = some(40);
    CHECK(ps::overlap(ps::region(&a), ps::region(&b)) ==
          ps::overlap(ps::region(&b), ps::region(&a)));
    const bool said = ps::overlap(ps::region(&a), ps::region(&b)), is = share(a, b);
    CHECK(said || !is);
    met += is;
    apart += !said;
    // a flat array against rows
    const size_t bytes = size_t(flat.cols) * 4;
    const ps::Region line = ps::region(flat.data, bytes);
    const ps_rows one = rows(reinterpret_cast<uintptr_t>(flat.data), 1, flat.cols, flat.cols, PS_F32);
    CHECK(ps::overlap(line, ps::region(&a)) || !share(one, a));
  }
  CHECK(met > 1000 && apart > 1000);
  return 0;
}

int streams() {
  const size_t bytes = ps::kStreamBytes;
  const uintptr_t at = 1 << 20;
  const auto dense = [&](size_t total, long long cols, int dtype) {
    return rows(at, (long long)(total / (size_t(cols) * ps::dtype_size(dtype))), cols, cols, dtype);
  };
  for (int dtype : {PS_F32, PS_F16, PS_BF16}) {
    const ps_rows whole = dense(bytes, 1024, dtype);
    CHECK(ps::streamed(&whole, whole.rows));
    CHECK(!ps::streamed(&whole, whole.rows - 1));  // slots that leave a row of it unwritten
    ps_rows range = whole;                         // the same rows, less of each
    range.cols = 1023;
    CHECK(!ps::streamed(&range, range.rows));
    // a narrow column range of a wide buffer: the span is 34 MB, what is written 0.3
    const ps_rows narrow = rows(at, 2100, 32, dtype == PS_F32 ? 4096 : 8192, dtype);
    CHECK(!ps::streamed(&narrow, narrow.rows));
    // slots of few tokens in a buffer for many, and more slots than rows
    const ps_rows spare = dense(8 * bytes, 4096, dtype);
    CHECK(!ps::streamed(&spare, 32));
    CHECK(ps::streamed(&spare, 1LL << 60));
  }
  return 0;
}

}  // namespace

int main() { return overlaps() || streams(); }
