// Host check of the paged cache's addressing: for page tables with good, bad
// and missing entries, every run that has an address lies whole in the pages of
// its sequence and KV head, bad entries have none, and offsets past 32 bits hold.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "nsa_paged_index.h"

int main() {
  int bad = 0;
  srand(1);
  for (int trial = 0; trial < 2000; ++trial) {
    const int P = 16 * (1 + rand() % 20), rpp = P / 16, mp = 1 + rand() % 9, Hkv = 1 + rand() % 5;
    const int D = 16 << (rand() % 4), np = trial % 3 == 0 ? 2000000000 : 1 + rand() % 50;
    std::vector<int32_t> row(mp);
    const int32_t odd[] = {-1, INT32_MIN, INT32_MAX, np, np - 1, 0};
    for (auto& x : row) x = rand() % 3 == 0 ? odd[rand() % 6] : rand() % np;
    const int hkv = rand() % Hkv;
    for (int run = -2; run < mp * rpp + 5; ++run) {
      const int64_t at = nsa::paged_run(row.data(), run, rpp, mp, np, Hkv, hkv, D);
      const bool in = run >= 0 && run < mp * rpp;
      const int page = in ? row[run / rpp] : -1;
      if (!in || page < 0 || page >= np) {
        if (at != -1) ++bad;
        continue;
      }
      const __int128 first = ((__int128)page * Hkv + hkv) * P * D, end = first + (__int128)P * D;
      if (at != (int64_t)(first + (__int128)(run % rpp) * 16 * D) || at < first || at + 16 * D > end) ++bad;
    }
    const int lens[] = {-1, INT32_MIN, INT32_MAX, 0, mp * P, mp * P - 1, rand() % (mp * P)};
    for (int len : lens) {
      const int pos = nsa::paged_new_pos(row.data(), len, P, mp, np);
      const bool in = len >= 0 && len < mp * P;
      const bool ok = in && row[len / P] >= 0 && row[len / P] < np;
      if (pos != (ok ? len : -1)) ++bad;
    }
  }
  printf("paged runs: %d wrong\n", bad);
  return bad != 0;
}
