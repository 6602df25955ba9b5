// operators_driver.cpp - the C entries of the paged-cache operators
// (sym_amd/csrc/attention.cpp) over the CPU stand-in of the HIP runtime, with
// kernels that only count their launches. Built and run by
// tests/test_attention_host.py; prints one line per check.
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstring>
#include <functional>
#include <mutex>
#include <thread>

#include "../../include/relx.h"
#include "attention.h"
#include "capi.h"
#include "hip_fake.h"
#include "runtime.h"

namespace relx {
namespace {
int g_launches = 0;
}
hipError_t tables_launch(TablesArgs, hipStream_t) { return ++g_launches, hipSuccess; }
int rotate_blocks(int, int64_t, int64_t) { return 1; }
int rotate_lanes(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : dim <= 256 ? 32 : 64; }
hipError_t rotate_launch(const RotateArgs &, int, int, hipStream_t) { return ++g_launches, hipSuccess; }
hipError_t attend_launch_f16(const AttendArgs &, const AttendPlan &, hipStream_t) { return ++g_launches, hipSuccess; }
hipError_t attend_launch_f16_i8(const AttendArgs &, const AttendPlan &, hipStream_t) { return ++g_launches, hipSuccess; }
hipError_t attend_launch_bf16(const AttendArgs &, const AttendPlan &, hipStream_t) { return ++g_launches, hipSuccess; }
hipError_t attend_launch_bf16_i8(const AttendArgs &, const AttendPlan &, hipStream_t) { return ++g_launches, hipSuccess; }
} // namespace relx

namespace {

relx_ctx *g_ctx;
int32_t g_int[64];
int64_t g_long[64];

// A call's error code, or "ok".
std::string tables() {
  relx_block_tables_args a{};
  a.starts = g_int;
  a.taken = g_int + 1;
  a.slots = g_long;
  a.positions = g_int + 2;
  a.page = 16;
  a.rows = 1;
  relx_err err;
  return relx_block_tables(g_ctx, &a, 0, &err) == RELX_OK ? "ok" : err.code;
}

// Whether `call` returns while another thread holds the context's mutex, as a
// transfer does until the GPU has done it.
std::string beside_a_transfer(const std::function<std::string()> &call) {
  std::atomic<bool> done{false};
  std::string result;
  std::unique_lock<std::mutex> transfer(g_ctx->ctx->mu);
  std::thread other([&] {
    result = call();
    done = true;
  });
  for (int i = 0; i < 1000 && !done; ++i) // ten seconds at most
    std::this_thread::sleep_for(std::chrono::milliseconds(10));
  const bool returned = done;
  transfer.unlock();
  other.join();
  return returned ? result : "waited";
}

void say(const char *what, const std::string &result) { std::printf("%s: %s\n", what, result.c_str()); }

} // namespace

int main() {
  fake_configure(nullptr);
  relx_err err;
  if (relx_ctx_create(0, -1, &g_ctx, &err) != RELX_OK)
    return 1;
  say("tables", tables());
  say("tables beside a transfer", beside_a_transfer(tables));
  say("launches", std::to_string(relx::g_launches));
  g_ctx->ctx->quarantined = true;
  say("tables of a quarantined context", tables());
  g_ctx->ctx->quarantined = false;
  if (relx_ctx_close(g_ctx, &err) != RELX_OK)
    return 1;
  fake_shutdown();
}
