// workspace_growth.cpp -- what a context allocates for split calls that grow a
// little at a time, as those over a cache that fills do, on a host-only build (TEST
// INFRASTRUCTURE ONLY; no GPU).  HIP is a handful of stubs: memory is a number.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <map>

#include "core_kernels.hpp"
#include "ctx.hpp"
#include "imq.h"
#include "imq_core.h"

namespace {

int allocations = 0, unsplit = 0;
size_t live = 0, largest_allowed = SIZE_MAX;
std::map<void*, size_t> memory;
uintptr_t next = 0x10000;
bool capturing = false;

[[noreturn]] void die(const char* what) {
  fprintf(stderr, "workspace_growth: %s (%d allocations, %zu bytes)\n", what, allocations, live);
  _Exit(4);
}

}  // namespace

extern "C" {
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) {
  if (capturing) die("an allocation under capture");
  if (n > largest_allowed) return hipErrorOutOfMemory;
  ++allocations;
  live += n;
  *p = reinterpret_cast<void*>(next);
  next += (n + 4095) / 4096 * 4096;
  memory[*p] = n;
  return hipSuccess;
}
hipError_t hipFree(void* p) {
  if (!memory.count(p)) die("freed what was not allocated");
  live -= memory[p];
  memory.erase(p);
  return hipSuccess;
}
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
  *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
}

namespace imq {
hipError_t launch_ln_mod(const void*, int, const float*, const float*, const int32_t*, int, void*,
                         int, int, int, float, float, hipStream_t) {
  return hipSuccess;
}
hipError_t launch_rope(const RopeArgs&, bool, int, hipStream_t) { return hipSuccess; }
AttnPlan attention_plan(const AttnArgs& a, int) {
  AttnPlan p{};
  p.splits = 2;
  p.bytes = (size_t)a.max_k * 1000;
  return p;
}
hipError_t use(const void* ws, size_t need) {
  if (!ws) {
    ++unsplit;
    return hipSuccess;
  }
  if (memory.at(const_cast<void*>(ws)) < need) die("a workspace that is too small");
  return hipSuccess;
}
hipError_t launch_attention(const AttnArgs&, const AttnPlan& plan, float* ws, int, hipStream_t) {
  return use(ws, plan.bytes);
}
size_t qgemm_split_bytes(int k, int, int, bool) { return (size_t)k * 1000; }
size_t qskinny_split_bytes(int k, int, int) { return (size_t)k * 1000; }
hipError_t launch_qgemm(const uint32_t*, const void*, const void*, const void*, void*, int k, int, int,
                        int, hipStream_t, SplitWs ws) {
  return use(ws.p, (size_t)k * 1000);
}
hipError_t launch_qskinny(const uint32_t*, const void*, const void*, const void*, void*, int k, int, int,
                          int, hipStream_t, SplitWs ws) {
  return use(ws.p, (size_t)k * 1000);
}
}  // namespace imq

namespace {

alignas(16) char mem[4096];

void attention(imq_ctx* ctx, int keys, hipStream_t st = nullptr) {
  imq_attention_args a{};
  a.q = a.k = a.v = mem;
  a.out = mem + 2048;
  a.q_row = a.out_row = 64, a.q_head = a.out_head = 64;
  a.k_row = a.v_row = 64, a.k_head = a.v_head = 64;
  a.n_seq = 1, a.heads = 1, a.kv_heads = 1, a.dim = 64, a.max_q = 1, a.max_k = keys;
  a.scale = 0.125f;
  a.dtype = IMQ_F16;
  if (imq_attention(ctx, &a, st) != IMQ_OK) die(imq_last_error(ctx));
}

void matmul(imq_ctx* ctx, int k, int m) {
  if (imq_qmm_t(ctx, reinterpret_cast<uint32_t*>(mem), mem, mem, mem, mem, k, 64, m, 64, 4, IMQ_F16, nullptr) != IMQ_OK)
    die(imq_last_error(ctx));
}

}  // namespace

int main() {
  int most = 0;
  for (int what = 0; what < 3; ++what) {
    imq_ctx ctx;
    ctx.cus = 256;
    allocations = 0;
    // 64 KB to 32 MB in steps of 64 KB, then down again.
    for (int k = 64; k <= 32768; k += 64) what == 0 ? attention(&ctx, k) : matmul(&ctx, k, what == 1 ? 8 : 40);
    for (int k = 32768; k > 64; k -= 6400) what == 0 ? attention(&ctx, k) : matmul(&ctx, k, what == 1 ? 8 : 40);
    most = std::max(most, allocations);
    if (allocations > 10) die("an allocation every few calls");
    if (live > 4 * (size_t)32768 * 1000) die("outgrown workspaces of several times the one in use");
  }
  if (live != 0) die("memory is left behind a context");
  if (unsplit != 0) die("a call ran unsplit");
  {
    // Memory for just what a call needs.
    imq_ctx ctx;
    ctx.cus = 256;
    largest_allowed = 5000 * 1000;
    attention(&ctx, 5000);
    if (unsplit != 0) die("unsplit where there is memory");
    attention(&ctx, 5001);
    if (unsplit != 1) die("no memory, and yet split");
    largest_allowed = SIZE_MAX;
    // A captured call that a smaller one has made room for.
    capturing = true;
    attention(&ctx, 5000);
    if (unsplit != 1) die("unsplit where there is room");
    attention(&ctx, 60000);
    if (unsplit != 2) die("captured without room, and yet split");
  }
  if (live != 0) die("memory is left behind a context");
  printf("workspace_growth: %d allocations\n", most);
  return 0;
}
