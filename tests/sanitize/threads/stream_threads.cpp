// stream_threads.cpp -- calls with a split workspace from several host threads,
// on a host-only build (TEST INFRASTRUCTURE ONLY; no GPU).
//
// A split call enqueues two kernels, the ranges and the join, which meet in the
// workspace of their stream.  The launchers here write down the order in which a
// stream gets them; no other user of the workspace may come between a call's two.
// HIP is a handful of stubs: memory is host memory that no kernel touches.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>
#include <thread>
#include <vector>

#include "core_kernels.hpp"
#include "ctx.hpp"
#include "imq.h"
#include "imq_core.h"

namespace {

std::atomic<int> allocations{0}, capturing{0}, calls{0}, unsplit{0};
std::mutex log_mu;
std::map<hipStream_t, std::vector<int>> order;  // of the split kernels: call i is 2 i, then 2 i + 1
std::map<const void*, hipStream_t> owner;       // of every workspace that was used

[[noreturn]] void die(const char* what) {
  fprintf(stderr, "stream_threads: %s\n", what);
  _Exit(4);
}

void enqueue(hipStream_t st, int what) {
  std::lock_guard<std::mutex> lk(log_mu);
  order[st].push_back(what);
}

// A call with a workspace of `need` bytes: its two kernels.
hipError_t two_kernels(hipStream_t st, const void* ws) {
  const int call = calls++;
  if (!ws) {
    ++unsplit;
    return hipSuccess;
  }
  {
    std::lock_guard<std::mutex> lk(log_mu);
    auto at = owner.emplace(ws, st).first;
    if (at->second != st) die("two streams use one workspace");
  }
  enqueue(st, 2 * call);
  std::this_thread::sleep_for(std::chrono::microseconds(50));  // long enough for the others
  enqueue(st, 2 * call + 1);
  return hipSuccess;
}

std::map<const void*, std::thread::id> per_thread;  // of the workspaces of threads' own streams

// Both streams' calls are between their kernels at once, or the wait gives up.
std::atomic<int> meeting{0};
std::atomic<bool> met{false};

}  // namespace

extern "C" {
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipMalloc(void** p, size_t n) {
  ++allocations;
  *p = malloc(n);
  return *p ? hipSuccess : hipErrorOutOfMemory;
}
hipError_t hipFree(void* p) {
  free(p);
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
// As many bytes as there are keys.
AttnPlan attention_plan(const AttnArgs& a, int) {
  AttnPlan p{};
  p.kernel = IMQ_ATTENTION_FEW;
  p.splits = a.max_k > 1 ? 2 : 1;
  p.bytes = a.max_k > 1 ? (size_t)a.max_k : 0;
  return p;
}
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, float* ws, int, hipStream_t st) {
  if ((plan.bytes > 0) != (ws != nullptr)) die("a plan without its workspace");
  if (a.max_q == 7) {  // the meeting of two streams
    ++meeting;
    for (int i = 0; i < 20000 && meeting < 2; ++i)
      std::this_thread::sleep_for(std::chrono::microseconds(100));
    if (meeting >= 2) met = true;
  }
  if (st == hipStreamPerThread) {
    std::lock_guard<std::mutex> lk(log_mu);
    const auto at = per_thread.emplace(ws, std::this_thread::get_id()).first;
    if (at->second != std::this_thread::get_id()) die("two threads' own streams use one workspace");
    return hipSuccess;
  }
  return two_kernels(st, ws);
}
size_t qgemm_split_bytes(int k, int, int, bool) { return (size_t)k; }
size_t qskinny_split_bytes(int k, int, int) { return (size_t)k; }
hipError_t launch_qgemm(const uint32_t*, const void*, const void*, const void*, void*, int, int, int,
                        int, hipStream_t st, SplitWs ws) {
  return two_kernels(st, ws.p);
}
hipError_t launch_qskinny(const uint32_t*, const void*, const void*, const void*, void*, int, int, int,
                          int, hipStream_t st, SplitWs ws) {
  return two_kernels(st, ws.p);
}
}  // namespace imq

namespace {

alignas(16) char mem[4096];
const auto kStream = reinterpret_cast<hipStream_t>(0x1000), kOther = reinterpret_cast<hipStream_t>(0x2000);

void attention(imq_ctx* ctx, hipStream_t st, int keys, int queries = 1) {
  imq_attention_args a{};
  a.q = a.k = a.v = mem;
  a.out = mem + 2048;
  a.q_seq = a.out_seq = 512, a.q_row = a.out_row = 64, a.q_head = a.out_head = 64;
  a.k_seq = a.v_seq = 1 << 20, a.k_row = a.v_row = 64, a.k_head = a.v_head = 64;
  a.n_seq = 1, a.heads = 1, a.kv_heads = 1, a.dim = 64, a.max_q = queries, a.max_k = keys;
  a.scale = 0.125f;
  a.dtype = IMQ_F16;
  if (imq_attention(ctx, &a, st) != IMQ_OK) die(imq_last_error(ctx));
}

// m: 8 rows take the few-row kernel, 40 the tiles.
void matmul(imq_ctx* ctx, hipStream_t st, int k, int m) {
  if (imq_qmm_t(ctx, reinterpret_cast<uint32_t*>(mem), mem, mem, mem, mem, k, 64, m, 64, 4, IMQ_F16, st) != IMQ_OK)
    die(imq_last_error(ctx));
}

void check_pairs() {
  for (const auto& s : order)
    for (size_t i = 0; i < s.second.size(); i += 2)
      if (s.second[i] % 2 != 0 || s.second[i + 1] != s.second[i] + 1) {
        fprintf(stderr, "stream_threads: kernels %d and %d of stream %p in a row\n", s.second[i], s.second[i + 1],
                (void*)s.first);
        _Exit(4);
      }
}

void threads() {
  imq_ctx ctx;
  ctx.cus = 256;
  std::vector<std::thread> all;
  for (int t = 0; t < 6; ++t)
    all.emplace_back([&ctx, t] {
      for (int i = 0; i < 40; ++i) {
        // Sizes that grow, so that the workspace does, under the other threads.
        if (t % 3 == 0) attention(&ctx, t < 5 ? kStream : kOther, 2 + 64 * i);
        else matmul(&ctx, t < 5 ? kStream : kOther, 512 + 64 * i, t % 3 == 1 ? 8 : 40);
      }
    });
  for (auto& t : all) t.join();
  check_pairs();
  if (unsplit != 0) die("a call ran unsplit");
  if (order[kStream].size() != 2 * 5 * 40 || order[kOther].size() != 2 * 40) die("calls are missing");
}

// A call on one stream does not wait for another stream's.
void streams() {
  imq_ctx ctx;
  ctx.cus = 256;
  std::thread a([&] { attention(&ctx, kStream, 100, 7); }), b([&] { attention(&ctx, kOther, 100, 7); });
  a.join(), b.join();
  if (!met) die("streams wait for each other");
}

// hipStreamPerThread is one handle for as many streams as there are threads.
void own_streams() {
  imq_ctx ctx;
  ctx.cus = 256;
  for (int round = 0; round < 2; ++round) {  // a thread's memory may be another one's afterwards
    std::thread a([&] { attention(&ctx, hipStreamPerThread, 100); attention(&ctx, hipStreamPerThread, 200); });
    std::thread b([&] { attention(&ctx, hipStreamPerThread, 100); attention(&ctx, hipStreamPerThread, 200); });
    a.join(), b.join();
    attention(&ctx, hipStreamPerThread, 100);
  }
  if (per_thread.size() != 5) die("threads' own streams have other than a workspace each");
}

// Where nothing may be allocated, calls run unsplit and leave no lock behind:
// few rows past 16 fall through to the tiles, which ask again.
void captured() {
  imq_ctx ctx;
  ctx.cus = 256;
  capturing = 1;
  unsplit = 0;
  attention(&ctx, kStream, 100, 1);
  matmul(&ctx, kStream, 512, 8);
  matmul(&ctx, kStream, 512, 24);
  matmul(&ctx, kStream, 512, 40);
  capturing = 0;
}

}  // namespace

int main() {
  threads();
  order.clear(), owner.clear();
  streams();
  owner.clear();
  captured();
  own_streams();
  printf("stream_threads: %d calls, %d allocations\n", calls.load(), allocations.load());
  return 0;
}
