// Host check of the overlap test of the attention layer's views
// (tensorrs_b200/csrc/heads.h): random small views against the bytes that they
// reach, and slices of one buffer along each of its dimensions.  Prints
//   random <pairs> <share a byte> <of these not seen> <apart and seen as such>
//   slices <pairs> <refused>
#include <cstdio>
#include <cstring>
#include <random>
#include <set>
#include <vector>

#include "heads.h"

using namespace trs;

static trs_view make(int dtype, std::vector<int64_t> shape, std::vector<int64_t> strides, int64_t offset) {
  trs_view v;
  std::memset(&v, 0, sizeof(v));
  v.data = reinterpret_cast<void*>(uintptr_t(1 << 20));
  v.storage_len = 1 << 20;
  v.dtype = dtype;
  v.ndim = (int)shape.size();
  for (int i = 0; i < v.ndim; ++i) {
    v.shape[i] = shape[i];
    v.strides[i] = strides[i];
  }
  v.offset = offset;
  return v;
}

static std::set<int64_t> bytes(const trs_view& v) {
  std::set<int64_t> s;
  const int64_t n = numel_of(v.shape, v.ndim), es = dtype_size(v.dtype);
  for (int64_t i = 0; i < n; ++i) {
    int64_t at = v.offset, r = i;
    for (int d = v.ndim - 1; d >= 0; --d) {
      at += r % v.shape[d] * v.strides[d];
      r /= v.shape[d];
    }
    for (int64_t b = 0; b < es; ++b) s.insert(at * es + b);
  }
  return s;
}

int main() {
  std::mt19937 g(1);
  auto pick = [&](int lo, int hi) { return lo + (int)(g() % (unsigned)(hi - lo + 1)); };
  int pairs = 0, share = 0, missed = 0, apart = 0;
  for (; pairs < 200000; ++pairs) {
    trs_view v[2];
    const int64_t common[4] = {pick(1, 40), pick(1, 40), pick(1, 12), pick(1, 3)};
    for (trs_view& x : v) {
      const int nd = pick(1, 4);
      std::vector<int64_t> shape, strides;
      for (int i = 0; i < nd; ++i) {
        shape.push_back(pick(0, 9) ? pick(1, 4) : 0);
        const int64_t s = pick(0, 2) ? common[pick(0, 3)] : pick(0, 30);
        strides.push_back(pick(0, 3) ? s : -s);
      }
      x = make(pick(0, 3) ? TRS_F32 : TRS_F64, shape, strides, 400 + pick(0, 60));
    }
    const std::set<int64_t> a = bytes(v[0]), b = bytes(v[1]);
    bool common_byte = false;
    for (int64_t x : a) common_byte = common_byte || b.count(x);
    const bool seen = heads_overlap(&v[0], &v[1]);
    if (seen != heads_overlap(&v[1], &v[0])) ++missed;
    if (common_byte) ++share;
    if (common_byte && !seen) ++missed;
    if (!common_byte && !seen) ++apart;
  }
  std::printf("random %d %d %d %d\n", pairs, share, missed, apart);

  // a buffer [B, T, H, D] with one dimension of 3 more, at every place; slices of
  // it of one, two or more entries
  int cases = 0, refused = 0;
  for (int place = 0; place < 5; ++place) {
    const int64_t dims[4] = {2, 5, 3, 8};
    int64_t shape[5];
    for (int i = 0, k = 0; i < 5; ++i) shape[i] = i == place ? 3 : dims[k++];
    int64_t strides[5], step = 1;
    for (int i = 4; i >= 0; --i) {
      strides[i] = step;
      step *= shape[i];
    }
    std::vector<int64_t> sh, st;
    for (int i = 0; i < 5; ++i)
      if (i != place) {
        sh.push_back(shape[i]);
        st.push_back(strides[i]);
      }
    for (int a = 0; a < 3; ++a)
      for (int b = 0; b < 3; ++b) {
        if (a == b) continue;
        for (int fewer = 0; fewer < 4; ++fewer) {  // the second slice shorter along one dimension
          std::vector<int64_t> sb = sh;
          sb[fewer] -= fewer ? 1 : 0;
          const trs_view x = make(TRS_F32, sh, st, a * strides[place]), y = make(TRS_F32, sb, st, b * strides[place]);
          ++cases;
          refused += heads_overlap(&x, &y);
        }
      }
  }
  std::printf("slices %d %d\n", cases, refused);
  return 0;
}
