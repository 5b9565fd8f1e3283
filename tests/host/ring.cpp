// The drains of dc_ring.h against a model of barriers that know a phase by its parity alone.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "dc_ring.h"

// A ring of S buffers: how many phases of each barrier are complete, which copies are in flight.
template <int S>
struct Ring {
  int done[S] = {};
  std::vector<int> flying;
  bool stuck = false;  // a wait that nothing would ever meet
  void land(size_t k) {
    done[flying[k] % S]++;
    flying.erase(flying.begin() + k);
  }
  // A wait: returns at once unless the phase under way has this parity; then the copy that ends it lands.
  void wait(int st, uint32_t parity) {
    if ((uint32_t)(done[st] & 1) != parity) return;
    for (size_t k = 0; k < flying.size(); k++)
      if (flying[k] % S == st) return land(k);
    stuck = true;
  }
  // Copies 0 .. landed - 1 have landed, landed .. issued - 1 fly but for those in `early`.
  Ring(int landed, int issued, unsigned early) {
    for (int i = 0; i < landed; i++) done[i % S]++;
    for (int i = landed; i < issued; i++) flying.push_back(i);
    for (int i = issued - 1; i >= landed; i--)
      if (early >> (i - landed) & 1) land(i - landed);
  }
};

static int fails = 0;
static void check(bool ok, const char* what, int a, int b, unsigned c) {
  if (!ok && fails++ < 20) printf("%s: %d %d early %x\n", what, a, b, c);
}

template <int S>
static bool phase_zero_rule_leaves_copies() {  // waiting for phase 0 of every stage (a planted mistake)
  for (int n = 1; n < 20; n++)
    for (int i = 0; i < n; i++) {
      const int issued = i + S < n ? i + S : n;
      Ring<S> r(i, issued, 0);
      for (int st = 0; st < S; st++)
        if (st < n) r.wait(st, 0);
      if (!r.flying.empty()) return true;
    }
  return false;
}

template <int S>
static void rings() {
  for (int n = 1; n < 30; n++)
    for (int i = 0; i <= n; i++) {
      // a warp that copies for itself and gave up on tile i
      const int issued = i + S < n ? i + S : n;
      for (unsigned early = 0; early < 1u << (issued - i); early++) {
        Ring<S> r(i, issued, early);
        dcr::drain_own<S>(i, n, [&](int st, uint32_t par) { r.wait(st, par); });
        check(r.flying.empty() && !r.stuck, "drain_own", n, i, early);
      }
    }
  for (int issued = 0; issued < 30; issued++) {
    // a copier whose last copies fly, in any state of the newest S
    const int landed = issued > S ? issued - S : 0;
    for (unsigned early = 0; early < 1u << (issued - landed); early++) {
      Ring<S> r(landed, issued, early);
      dcr::drain<S>(issued, [&](int st, uint32_t par) { r.wait(st, par); });
      check(r.flying.empty() && !r.stuck, "drain", issued, 0, early);
    }
  }
  check(phase_zero_rule_leaves_copies<S>(), "the model misses the planted mistake", S, 0, 0);
}

int main() {
  rings<3>();
  rings<5>();
  rings<6>();
  rings<8>();
  return fails ? 1 : 0;
}
