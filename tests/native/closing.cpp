// Closing of handles over a runtime of two devices, without a GPU: the caller's device is the same behind each call, memory is
// freed on the session's, and pages and logits that any stream may read only after the whole device was waited for.
// Exit status 0 and "ok" when every check holds.
#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <set>

#include "../../include/rstr_hip.h"
#include "../../pretrained-rstr_amd/csrc/kernels.h"

static int g_device = 0, g_freed = 0, g_astray = 0, g_unwaited = 0, g_work = 0;
static std::set<void*> g_blocks;

static hipError_t take(void** p, size_t n) { return *p = calloc(1, n ? n : 1), g_blocks.insert(*p), hipSuccess; }
static hipError_t give(void* p) {
  if (!p) return hipSuccess;
  if (!g_blocks.erase(p)) printf("a free of memory that is not allocated\n"), exit(1);
  free(p);
  g_freed++;
  g_astray += g_device != 1;
  g_unwaited += g_work;
  return hipSuccess;
}

extern "C" {
hipError_t hipMalloc(void** p, size_t n) { return take(p, n); }
hipError_t hipHostMalloc(void** p, size_t n, unsigned) { return take(p, n); }
hipError_t hipFree(void* p) { return give(p); }
hipError_t hipHostFree(void* p) { return give(p); }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { return memmove(d, s, n), hipSuccess; }
hipError_t hipMemset(void* d, int v, size_t n) { return memset(d, v, n), hipSuccess; }
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t) { return memset(d, v, n), hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = g_device, hipSuccess; }
hipError_t hipSetDevice(int d) { return g_device = d, hipSuccess; }
hipError_t hipGetDeviceCount(int* n) { return *n = 2, hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { return *s = reinterpret_cast<hipStream_t>(&g_device), hipSuccess; }
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return g_work = 0, hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return *e = reinterpret_cast<hipEvent_t>(&g_device), hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned) { return *e = reinterpret_cast<hipEvent_t>(&g_device), hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
}

namespace rstr {
static char g_scratch[64];
hipError_t static_scratch_address(void** p) { return *p = g_scratch, hipSuccess; }
hipError_t launch_gen_linear(hipStream_t, const QTensor&, int, int, int, uint64_t, const float*) { return hipSuccess; }
hipError_t launch_gen_f32(hipStream_t, float*, int64_t, uint64_t, double, double, double) { return hipSuccess; }
size_t attn_tab_words(const AttnGeom& g, int max_items) { return 8 * (size_t)g.batch + 4 * (size_t)max_items; }
int qgemm_splits(int, int, int) { return 1; }
int qgemm_head_splits(int, int, int, int) { return 1; }
bool qgemm_act_fused(int, int) { return false; }
bool attn_fuses_qkv(const AttnGeom&, int) { return false; }
bool attn_direct_out(const AttnGeom&, int) { return false; }
int argmax_segments(int, int) { return 1; }
void pool_shared(rstr_pool*);
}  // namespace rstr

static rstr_session* g_s;
#define CHECK(x)                                                                 \
  do {                                                                           \
    if (!(x)) {                                                                  \
      printf("line %d: %s (%s)\n", __LINE__, #x, g_s ? rstr_last_error(g_s) : ""); \
      return 1;                                                                  \
    }                                                                            \
  } while (0)
#define CLOSES(call)                                                 \
  do {                                                               \
    const int before = g_freed;                                      \
    g_device = 0;                                                    \
    g_work = 1; /* on a stream of the caller's */                    \
    CHECK((call) == RSTR_OK);                                        \
    CHECK(g_device == 0 && g_astray == 0 && g_freed > before);       \
  } while (0)

int main() {
  rstr_model_desc d{};
  d.n_layers = 1;
  d.d_model = d.d_ff = 128;
  d.n_q = 8;
  d.n_kv = 1;
  d.head_dim = 128;
  d.vocab = 512;
  d.weight_bits = 4;
  d.eps = 1e-6f;
  d.attn_scale = 0.1f;
  d.rope_global = d.rope_local = 1e4;
  rstr_model* m = nullptr;
  rstr_pool* p = nullptr;
  rstr_decoder* dec = nullptr;
  CHECK(rstr_session_open(1, &g_s) == RSTR_OK);
  CHECK(rstr_model_bind_synthetic(g_s, &d, 1, &m) == RSTR_OK);
  CHECK(rstr_pool_open(m, 16, 8, &p) == RSTR_OK);
  rstr::pool_shared(p);  // as an operator on device arrays, or a lent address, leaves it
  CHECK(rstr_decoder_open(m, p, 2, 4, 32, 16, &dec) == RSTR_OK);
  CLOSES(rstr_decoder_close(dec));
  CHECK(g_unwaited == 0);
  CLOSES(rstr_pool_close(p));
  CHECK(g_unwaited == 0);
  CLOSES(rstr_model_close(m));
  g_device = 0;
  CHECK(rstr_session_close(g_s) == RSTR_OK && g_device == 0 && g_blocks.empty());
  printf("ok\n");
  return 0;
}
