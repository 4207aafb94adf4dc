// How the 8-bit products are cut up, without a GPU: the plan of gemm_q8.cu and what its CTAs ask for.
#include "../p2p_b200/csrc/gemm_q8.cu"

// out: 1 where pairs of CTAs take the call; channels and tokens of a tile, CTAs of its k, steps of 128 codes
// in a stage, stages of a tile, tiles, stages of the ring, bytes of shared memory, columns of TMEM; and of
// pairs of CTAs: items.
extern "C" __attribute__((visibility("default"))) void host_plan(int m, int n, int k, int gate,
                                                                 int num_sms, int room, int64_t* out) {
  using namespace p2p;
  const int G = gate ? 2 : 1;
  const Choice c = choose(m, n, k, G, num_sms, room);
  out[0] = c.wide;
  if (c.wide) {
    const WideItems w = wide_items(m, n, G, num_sms / 2);
    out[1] = w.whole;
    out[2] = w.items;
    return;
  }
  const NarrowPlan& p = c.plan;
  const int64_t tiles = (int64_t(n) + p.rows - 1) / p.rows * ((m + p.tokens - 1) / p.tokens);
  const NarrowRoom r = narrow_room(p, G, tiles, num_sms);
  const int64_t v[] = {p.rows, p.tokens, p.split, p.chunks, p.steps, tiles, r.stages, r.smem, r.cols};
  for (int i = 0; i < 9; ++i) out[1 + i] = v[i];
}
