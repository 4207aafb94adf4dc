// The search for a row's sequence (kv_view.cuh), run on the host with the 32 lanes one after the
// other: reads lines "nseq row_start[0 .. nseq] n rows" and prints the sequence of each row.
#include <cstdio>
#include <vector>

#include "kv_view.cuh"

int main() {
  int nseq, n;
  while (std::scanf("%d", &nseq) == 1) {
    std::vector<int32_t> start(nseq + 1);
    for (auto& s : start)
      if (std::scanf("%d", &s) != 1) return 1;
    if (std::scanf("%d", &n) != 1) return 1;
    for (int i = 0; i < n; ++i) {
      long long r;
      if (std::scanf("%lld", &r) != 1) return 1;
      std::printf("%d ", p2p::find_seq(start.data(), nseq, r, [](auto f) {
                    int c = 0;
                    for (int lane = 0; lane < 32; ++lane) c += f(lane) ? 1 : 0;
                    return c;
                  }));
    }
    std::printf("\n");
  }
  return 0;
}
