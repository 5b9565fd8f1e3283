// The checks of strided buffers in dc_span.h against all their elements' addresses.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "dc_span.h"

using namespace dcc;

static int fails = 0;
static void check(bool ok, const char* what) {
  if (!ok && fails++ < 20) printf("%s\n", what);
}
static void places(const std::vector<Dim>& d, size_t k, int64_t at, std::vector<int64_t>& out) {
  if (k == d.size()) return out.push_back(at);
  for (int64_t i = 0; i < d[k].n; i++) places(d, k + 1, at + i * d[k].stride, out);
}
static bool distinct(const std::vector<Dim>& d, int64_t other = -1) {
  std::vector<int64_t> at;
  places(d, 0, 0, at);
  if (other >= 0) places(d, 0, other, at);
  return std::set<int64_t>(at.begin(), at.end()).size() == at.size();
}

int main() {
  // random strides: what passes has distinct elements
  srand(1);
  int passed = 0, refused = 0;
  for (int k = 0; k < 200000; k++) {
    Dim d[3];
    for (Dim& x : d) x = {1 + rand() % 4, rand() % 30};
    const bool ok = apart({d[0], d[1], d[2]});
    (ok ? passed : refused)++;
    check(!ok || distinct({d[0], d[1], d[2]}), "apart passes elements that coincide");
    // and two such buffers
    const int64_t step = rand() % 60;
    static int16_t base[400];
    const Span a = span(base, 2, {d[0], d[1], d[2]}), b = span(base + step, 2, {d[0], d[1], d[2]});
    check(!ok || !twins_apart(a, b, 2, {d[0], d[1], d[2]}, {d[0], d[1], d[2]}) || distinct({d[0], d[1], d[2]}, step),
          "twins_apart passes elements that coincide");
  }
  check(passed > 1000 && refused > 1000, "both answers are drawn");

  // layouts in use: sequences 3, tokens 8, heads 2, channels 64
  static float base[40000];
  const int64_t S = 3, T = 8, H = 2, D = 64;
  auto both = [&](Dim s, Dim t, Dim h, int64_t step) {
    const Span a = span(base, 4, {s, t, h, {D, 1}}), b = span(base + step, 4, {s, t, h, {D, 1}});
    return apart({s, t, h, {D, 1}}) && twins_apart(a, b, 4, {s, t, h, {D, 1}}, {s, t, h, {D, 1}}) &&
           twins_apart(b, a, 4, {s, t, h, {D, 1}}, {s, t, h, {D, 1}});
  };
  check(both({S, T * H * D}, {T, H * D}, {H, D}, S * T * H * D), "one after the other");
  check(both({S, 2 * T * H * D}, {T, 2 * H * D}, {H, 2 * D}, D), "side by side in a head");
  check(both({S, 2 * T * H * D}, {T, 2 * H * D}, {H, D}, H * D), "side by side in a token");
  check(both({S, 2 * T * H * D}, {T, H * D}, {H, D}, T * H * D), "side by side in a sequence");
  check(both({S, 2 * T * D}, {T, 2 * D}, {H, S * 2 * T * D}, D), "head-major");
  check(both({1, 0}, {T, 2 * H * D}, {H, 2 * D}, D), "one sequence, whatever its stride");
  check(both({S, (T + 5) * H * D}, {T, H * D}, {H, D}, S * (T + 5) * H * D), "more room than tokens");
  // and what is refused
  check(!both({S, T * H * D}, {T, H * D}, {H, D}, 0), "the same buffer");
  check(!both({S, T * H * D}, {T, H * D}, {H, D}, H * D), "a token further");
  check(!both({S, 2 * T * H * D}, {T, 2 * H * D}, {H, 2 * D}, D - 1), "one channel less than a row");
  check(!apart({{S, 0}, {T, H * D}, {H, D}, {D, 1}}), "expanded over sequences");
  check(!apart({{S, T * H * D}, {T, H * D}, {H, 0}, {D, 1}}), "expanded over heads");
  check(!apart({{S, T * H * D}, {T, D}, {H, D}, {D, 1}}), "tokens as near as heads");
  check(!apart({{T, 1}, {D, 1}}), "a sliding window");
  check(apart({{0, 0}, {T, 0}}), "no elements");
  const Span a = span(base, 4, {{T, 2 * D}, {D, 1}}), b = span(base + D, 4, {{T, D}, {D, 1}});
  check(!twins_apart(a, b, 4, {{T, 2 * D}, {D, 1}}, {{T, D}, {D, 1}}), "other strides in the same span");
  const Span c = span((char*)base + 2, 4, {{T, 2 * D}, {D, 1}});
  check(!twins_apart(a, c, 4, {{T, 2 * D}, {D, 1}}, {{T, 2 * D}, {D, 1}}), "half an element further");
  return fails ? 1 : 0;
}
