// The address arithmetic of a ragged chunk over a KV cache (kv_view.cuh), run on the host: reads
// cases from stdin and prints, per position, the row the kernels would touch or -1.
//   in:  table? kv_rows shift max_blocks past row0 row1 n_rows max_len offset, then max_blocks pages
//   out: ok, then a row per position past .. past + len - 1 (only when ok)
#include <cstdio>
#include <vector>

#include "kv_view.cuh"

int main() {
  long long paged, kv_rows, shift, max_blocks, past, r0, r1, n_rows, max_len, offset;
  while (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld %lld", &paged, &kv_rows, &shift,
                    &max_blocks, &past, &r0, &r1, &n_rows, &max_len, &offset) == 10) {
    std::vector<int32_t> table(max_blocks);
    for (auto& t : table)
      if (std::scanf("%d", &t) != 1) return 1;
    const int32_t p = int32_t(past), off = int32_t(offset), rs[2] = {int32_t(r0), int32_t(r1)};
    p2p::KvView c{};
    c.kv_rows = kv_rows;
    c.offsets = &off;
    c.table = paged ? table.data() : nullptr;
    c.max_blocks = int32_t(max_blocks);
    c.shift = int32_t(shift);
    const p2p::ChunkIndex x{&p, rs, 1, n_rows, int32_t(max_len)};
    const p2p::SeqSpan s = p2p::seq_span(c, x, 0);
    std::printf("%d", s.ok ? 1 : 0);
    for (int j = 0; s.ok && j < s.len; ++j)
      std::printf(" %lld", static_cast<long long>(p2p::kv_row(c, 0, s.past + j)));
    std::printf("\n");
  }
  return 0;
}
