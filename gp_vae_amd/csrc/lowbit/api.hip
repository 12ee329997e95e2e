// api.hip — library-wide pieces of the low-bit C ABI: error string, version, sizes of the formats.
#include "lowbit.hpp"

namespace gpvae_lb {
static thread_local char g_err[512] = "";
void set_error(const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
}
}  // namespace gpvae_lb

using namespace gpvae_lb;

extern "C" int gpvae_lowbit_abi_version(void) { return GPVAE_LOWBIT_ABI_VERSION; }
extern "C" const char *gpvae_lowbit_last_error(void) { return g_err; }
extern "C" int64_t gpvae_w4_code_bytes(int64_t K, int64_t N) { return K < 1 || N < 1 ? 0 : w4_kb(K) * w4_np(N) * 16; }
extern "C" int64_t gpvae_w4_exp_bytes(int64_t K, int64_t N) { return K < 1 || N < 1 ? 0 : w4_kb(K) * w4_np(N) / 2; }
extern "C" int64_t gpvae_q8_code_bytes(int64_t M, int64_t K) { return M < 1 || K < 1 ? 0 : q8_mb(M) * q8_kp(K) * 8; }
extern "C" int64_t gpvae_q8_exp_bytes(int64_t M, int64_t K) { return M < 1 || K < 1 ? 0 : q8_mb(M) * q8_kp(K) / 8; }
