// The host side of the 8-bit layer operators without a GPU: q8_api.cu with stand-ins for the context and
// the launchers, which count.  Its C entry points are called with made-up addresses.
#include "../p2p_b200/csrc/q8_api.cu"

#include <string>

static std::string g_message;
static int g_launches;

namespace p2p {
int ctx_device(const p2p_ctx*) { return 0; }
int ctx_num_sms(const p2p_ctx*) { return 148; }
int32_t debug_wait_deficit() { return 0; }
int32_t* ctx_dev_err(const p2p_ctx*) { return nullptr; }
p2p_status ctx_fail(p2p_ctx*, p2p_status s, const char* msg) {
  g_message = msg;
  return s;
}
cudaError_t launch_rows_q8(const RowsQ8Args&, int, int, cudaStream_t) {
  ++g_launches;
  return cudaSuccess;
}
cudaError_t launch_read_q8(const ReadQ8Args&, int, cudaStream_t) {
  ++g_launches;
  return cudaSuccess;
}
cudaError_t launch_gemm_q8(const GemmQ8Args&, int, int, cudaStream_t) {
  ++g_launches;
  return cudaSuccess;
}
}  // namespace p2p

extern "C" __attribute__((visibility("default"))) int host_launches() { return g_launches; }
extern "C" __attribute__((visibility("default"))) const char* host_message() {
  return g_message.c_str();
}
