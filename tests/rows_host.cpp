// rows_overlap (rows.h) on the host: reads lines "a pitch width b pitch width n", prints 0 or 1.
#include <cstdio>

#include "rows.h"

int main() {
  long long a, pa, wa, b, pb, wb, n;
  while (std::scanf("%lld %lld %lld %lld %lld %lld %lld", &a, &pa, &wa, &b, &pb, &wb, &n) == 7)
    std::printf("%d\n", p2p::rows_overlap(reinterpret_cast<void*>(a), pa, wa,
                                          reinterpret_cast<void*>(b), pb, wb, n)
                            ? 1
                            : 0);
  return 0;
}
