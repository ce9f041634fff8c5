// A group's arguments as its manifest describes them, and the checks that a
// launch's pass before anything runs.  No HIP in here: what a launch accepts
// does not depend on the device.
#pragma once
#include <algorithm>
#include <cstddef>
#include <cstdint>
#include <sstream>
#include <string>
#include <utility>
#include <vector>

// element size of a manifest element type name (i1 is one byte)
inline int elemSize(const std::string &e) {
  if (e == "f64" || e == "i64" || e == "index") return 8;
  if (e == "f32" || e == "i32") return 4;
  if (e == "f16" || e == "bf16" || e == "i16") return 2;
  return 1;
}

struct Buf {
  std::string elem;
  std::vector<int64_t> shape;
};

struct GroupArgs {
  std::string func;
  bool rowsDyn = false; // the row count comes with the launch (-1 in the shapes)
  bool rowsZero = false; // a launch of no rows has results to write (manifest `rows_zero 1`)
  int64_t maxRows = 0; // launch-time rows that the group takes at most (manifest `max_rows`; 0: any number)
  uint64_t wsBytes = 0;
  bool wsZero = false; // zero when first used, and what a launch leaves there the next one reads
  std::vector<std::string> paramRoles;
  std::vector<Buf> paramBufs, resultBufs;
  std::vector<int> resultTied;
  std::vector<int> apart;                 // parameters that no destination may overlap
  std::vector<int> inplace;               // ones that it may be, but overlap in no other way
  std::vector<std::pair<int, int>> align; // parameter, bytes it has to start on

  // Takes a manifest line of these; false: the key is another's.  A malformed
  // line leaves the stream failed.
  bool line(const std::string &key, std::istringstream &is) {
    if (key == "apart" || key == "inplace") {
      for (int i; is >> i;) (key == "apart" ? apart : inplace).push_back(i);
      is.clear();
    } else if (key == "align") {
      int i = -1, bytes = 0;
      is >> i >> bytes;
      if (i < 0 || bytes <= 0) is.setstate(std::ios::failbit);
      align.push_back({i, bytes});
    } else if (key == "workspace") {
      int z = 0;
      is >> wsBytes >> z;
      wsZero = z != 0;
    } else if (key == "rows_zero") {
      int z = 0;
      is >> z;
      rowsZero = z != 0;
    } else if (key == "max_rows") {
      is >> maxRows;
      if (maxRows <= 0) is.setstate(std::ios::failbit);
    } else if (key == "param" || key == "result") {
      int i, tied = -1, rank = 0;
      std::string role;
      Buf b;
      is >> i;
      if (key == "param") is >> role;
      else is >> tied;
      is >> b.elem >> rank;
      for (int d = 0; d < rank && is; ++d) { int64_t x; is >> x; b.shape.push_back(x); }
      if (key == "param") { paramRoles.push_back(role); paramBufs.push_back(b); }
      else { resultTied.push_back(tied); resultBufs.push_back(b); }
    } else {
      return false;
    }
    return true;
  }

  // After the manifest's last line: what the overlap check needs of it, so
  // that a launch only adds and compares (names compared and shapes multiplied
  // at every launch made a call of few rows 0.4 us longer).  False: more
  // arguments than a launch passes.
  bool prepare() {
    spans.clear();
    pairs.clear();
    if (apart.empty() && inplace.empty()) return true;
    auto at = [&](bool result, size_t i) {
      for (size_t s = 0; s < spans.size(); ++s)
        if (spans[s].index == i && spans[s].result == result) return s;
      const Buf &b = result ? resultBufs[i] : paramBufs[i];
      Span sp;
      sp.result = result;
      sp.index = i;
      sp.bytes = (uint64_t)elemSize(b.elem);
      for (const int64_t d : b.shape) {
        if (d < 0) sp.rows = true;
        else sp.bytes *= (uint64_t)d;
      }
      spans.push_back(sp);
      return spans.size() - 1;
    };
    std::vector<size_t> written, kept;
    for (size_t i = 0; i < paramRoles.size(); ++i)
      if (paramRoles[i] != "in" && paramRoles[i] != "scalar") written.push_back(at(false, i));
    for (size_t i = 0; i < resultTied.size(); ++i)
      if (resultTied[i] < 0) written.push_back(at(true, i));
    auto tensor = [&](int j) { return j >= 0 && (size_t)j < paramBufs.size() && paramRoles[j] != "scalar"; };
    auto add = [&](size_t a, size_t b, bool same) {
      for (const Pair &p : pairs)
        if ((p.a == a && p.b == b) || (p.a == b && p.b == a)) return;
      if (a != b) pairs.push_back({a, b, same});
    };
    for (const size_t a : written) {
      for (const int j : apart)
        if (tensor(j)) add(a, at(false, (size_t)j), false);
      for (const size_t b : written) add(a, b, false);
      for (const int j : inplace)
        if (tensor(j)) add(a, at(false, (size_t)j), true);
    }
    return spans.size() <= MAX_SPANS;
  }

  // Why a launch's arguments are refused, empty where they are not.
  std::string check(const uint64_t *params, size_t nparams, void *const *results, size_t nresults, int64_t rows) const {
    if (nparams != paramRoles.size())
      return "group @" + func + " takes " + std::to_string(paramRoles.size()) + " arguments, got " + std::to_string(nparams);
    if (nresults != resultTied.size())
      return "group @" + func + " has " + std::to_string(resultTied.size()) + " results, got " + std::to_string(nresults);
    if (nparams && !params) return "null params array";
    if (maxRows && rows > maxRows) return "group @" + func + " takes at most " + std::to_string(maxRows) + " rows a launch, got " + std::to_string(rows);
    // (a tensor of no rows has no address)
    auto empty = [&](const std::vector<Buf> &bufs, size_t i) {
      return rows == 0 && i < bufs.size() && std::count(bufs[i].shape.begin(), bufs[i].shape.end(), int64_t(-1)) != 0;
    };
    for (size_t i = 0; i < nparams; ++i)
      if (params[i] == 0 && paramRoles[i] != "scalar" && !empty(paramBufs, i))
        return "null device pointer for argument " + std::to_string(i);
    for (size_t i = 0; i < nresults; ++i)
      if (resultTied[i] < 0 && (!results || (!results[i] && !empty(resultBufs, i))))
        return "null device pointer for result " + std::to_string(i);
    if (!pairs.empty()) {
      uint64_t lo[MAX_SPANS], hi[MAX_SPANS];
      for (size_t s = 0; s < spans.size(); ++s) {
        const Span &sp = spans[s];
        const uint64_t n = sp.bytes * (sp.rows ? (uint64_t)rows : 1);
        const uint64_t at = sp.result ? (uint64_t)(uintptr_t)results[sp.index] : params[sp.index];
        lo[s] = n ? at : UINT64_MAX; // (nothing overlaps an empty one)
        hi[s] = n ? at + n : 0;
      }
      for (const auto &p : pairs)
        if (lo[p.a] < hi[p.b] && lo[p.b] < hi[p.a] && !(p.same && lo[p.a] == lo[p.b] && hi[p.a] == hi[p.b]))
          return spans[p.a].name() + " of @" + func + " is written and overlaps " + spans[p.b].name();
    }
    for (const auto &a : align)
      if ((size_t)a.first < nparams && params[a.first] % (uint64_t)a.second)
        return "argument " + std::to_string(a.first) + " of @" + func + " does not start on " + std::to_string(a.second) + " bytes";
    return {};
  }

  // Why a caller's workspace is refused: zeroed ones hold 64-bit words, of the
  // others 16 bytes a lane are read and written.
  std::string checkWorkspace(const void *ws) const {
    const uintptr_t on = wsZero ? 8 : 16;
    if (!wsBytes || (uintptr_t)ws % on == 0) return {};
    return "a workspace of group @" + func + " has to start on " + std::to_string(on) + " bytes";
  }

private:
  static constexpr size_t MAX_SPANS = 64;
  struct Span {
    bool result = false; // of a buffer of its own, not one written into an argument
    size_t index = 0;
    bool rows = false; // `bytes` are a row's
    uint64_t bytes = 0;
    std::string name() const { return (result ? "result " : "argument ") + std::to_string(index); }
  };
  std::vector<Span> spans;
  struct Pair {
    size_t a, b; // a written span, one that it may not overlap
    bool same;   // unless the two are one buffer
  };
  std::vector<Pair> pairs;
};
