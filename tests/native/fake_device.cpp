// The host side of the operators on device arrays without a GPU: sessions
// that need none, allocations that can be made to fail, and launches that are
// only counted, so that a refusal can be seen to come before any device work.
#include <hip/hip_runtime.h>

#include <cstdlib>
#include <string>

#include "../../pretrained-rstr_amd/csrc/kv4.h"
#include "../../pretrained-rstr_amd/csrc/session.h"

static std::string g_open;
static int g_launches = 0, g_blocks = 0, g_fail_alloc = 0, g_device = 0;
static hipStream_t g_stream = nullptr;

int rstr::fail(rstr_session* s, int code, const std::string& msg) { return (s ? s->err : g_open) = msg, code; }
hipError_t rstr::device_alloc(void** p, size_t n) {
  if (g_fail_alloc) return hipErrorOutOfMemory;
  *p = malloc(n < (1u << 20) ? n + 1 : 1u << 20);
  g_blocks++;
  return hipSuccess;
}
static hipError_t launched(hipStream_t st) { return g_stream = st, g_launches++, hipSuccess; }
hipError_t rstr::launch_kv4_append(hipStream_t st, const Kv4Layer&, int, int, const Rows&, const Rows&, const int32_t*) { return launched(st); }
hipError_t rstr::launch_kv4_read(hipStream_t st, const Kv4Layer&, int, int, const int32_t*, const Rows&, const Rows&) { return launched(st); }
size_t rstr::kv4_attn_workspace(int, int, int, int, int) { return 64; }
hipError_t rstr::launch_kv4_attn(hipStream_t st, int, const Kv4Attn&) { return launched(st); }
hipError_t rstr::launch_step_maps(hipStream_t st, const StepMaps&) { return launched(st); }
size_t rstr::verify_workspace(int, int, int) { return 64; }
hipError_t rstr::launch_verify(hipStream_t st, int, const Verify&) { return launched(st); }

extern "C" {
int rstr_session_open(int32_t device, rstr_session** out) {
  *out = new rstr_session();
  (*out)->device = device;
  (*out)->stream = (hipStream_t)0x5e55;
  return 0;
}
int rstr_session_close(rstr_session* s) { return delete s, 0; }
const char* rstr_last_error(const rstr_session* s) { return s->err.c_str(); }
const char* rstr_open_error(void) { return g_open.c_str(); }
int fake_launches(void) { return g_launches; }
int fake_blocks(void) { return g_blocks; }
void* fake_stream(void) { return g_stream; }
int fake_device(int set) { return set >= 0 ? g_device = set : g_device; }
void fake_fail_alloc(int on) { g_fail_alloc = on; }

hipError_t hipGetDevice(int* d) { return *d = g_device, hipSuccess; }
hipError_t hipSetDevice(int d) { return g_device = d, hipSuccess; }
hipError_t hipMemsetAsync(void*, int, size_t, hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize() { return hipSuccess; }
hipError_t hipFree(void* p) { return free(p), g_blocks--, hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "error"; }
}
