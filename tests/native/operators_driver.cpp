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
#include <set>
#include <string>
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

// norm and rotation into a result of these strides, dims of 8
std::string rotate(int64_t rows, int64_t row, int64_t heads, int64_t head) {
  relx_rotation r{};
  r.positions = g_int;
  r.rows = rows;
  r.heads = heads;
  r.dim = 8;
  r.bits = 16;
  relx_heads x{g_long, heads * 8, 8}, y{g_long, row, head};
  relx_err err;
  const std::string forward = relx_norm_rotate(g_ctx, &r, &x, nullptr, &y, nullptr, 0, &err) == RELX_OK ? "ok" : err.code;
  const std::string back = relx_norm_rotate_backward(g_ctx, &r, &x, nullptr, &x, nullptr, &y, nullptr, nullptr, nullptr,
                                                     nullptr, 0, 0, &err) == RELX_OK
                               ? "ok"
                               : err.code;
  return forward == back ? forward : forward + " and " + back;
}

// and by brute force
std::string rotate_walked(int64_t rows, int64_t row, int64_t heads, int64_t head) {
  std::set<int64_t> seen;
  for (int64_t r = 0; r < rows; ++r)
    for (int64_t h = 0; h < heads; ++h)
      for (int64_t d = 0; d < 8; ++d)
        if (!seen.insert(r * row + h * head + d).second)
          return "invalid_argument";
  return "ok";
}

// the two over all small strides
std::string rotate_everywhere() {
  int wrong = 0;
  for (int64_t rows = 1; rows < 6; ++rows)
    for (int64_t heads = 1; heads < 6; ++heads)
      for (int64_t row = 0; row < 60; row += 3)
        for (int64_t head = 0; head < 60; ++head)
          wrong += rotate(rows, row, heads, head) != rotate_walked(rows, row, heads, head);
  return std::to_string(wrong);
}

// one row into a cache of two pages of four slots of three heads
std::string append(int64_t page, int64_t slot, int64_t head) {
  relx_rotation r{};
  r.positions = g_int;
  r.rows = 1;
  r.kv_heads = 3;
  r.dim = 8;
  r.bits = 16;
  relx_heads x{g_long, 24, 8};
  relx_cache c{g_long, 96, 24, 8, g_long, page, slot, head, nullptr, nullptr, 2, 4, 3, 8, 0, 16};
  relx_err err;
  return relx_norm_rotate_append(g_ctx, &r, nullptr, &x, &x, nullptr, g_long, &c, 0, &err) == RELX_OK ? "ok" : err.code;
}

// heads of 512 of each kind
std::string rotate_wide(int64_t heads, bool cache) {
  relx_rotation r{};
  r.positions = g_int;
  r.rows = 1;
  r.heads = r.kv_heads = heads;
  r.dim = 512;
  r.bits = 16;
  relx_heads x{g_long, heads * 512, 512};
  relx_cache c{g_long, heads * 512, heads * 512, 512, g_long, heads * 512, heads * 512, 512, nullptr, nullptr, 1, 1,
               heads,  512,         0,           16};
  relx_err err;
  const int rc = cache ? relx_norm_rotate_append(g_ctx, &r, &x, &x, &x, &x, g_long, &c, 0, &err)
                       : relx_norm_rotate(g_ctx, &r, &x, &x, &x, &x, 0, &err);
  return rc == RELX_OK ? "ok" : err.code;
}

// one row of `requests` requests
std::string attend_many(int64_t requests) {
  relx_tree_attention_args a{};
  a.q = a.out = {g_long, 8, 8};
  a.cache = {g_long, 8, 8, 8, g_long, 8, 8, 8, nullptr, nullptr, 1, 1, 1, 8, 0, 16};
  a.rows = a.heads = 1;
  a.requests = requests;
  a.cached = a.starts = g_int;
  alignas(16) static char room[16];
  a.workspace = room;
  a.workspace_bytes = INT64_MAX;
  a.bits = 16;
  a.scale = 1.0;
  relx_err err;
  return relx_tree_attention(g_ctx, &a, 0, &err) == RELX_OK ? "ok" : err.code;
}

std::string attend(int64_t rows, int64_t row, int64_t heads, int64_t head) {
  relx_tree_attention_args a{};
  a.q = {g_long, heads * 8, 8};
  a.out = {g_long, row, head};
  a.cache = {g_long, 96, 24, 8, g_long, 96, 24, 8, nullptr, nullptr, 2, 4, heads, 8, 0, 16};
  a.rows = rows;
  a.heads = heads;
  a.bits = 16;
  a.scale = 1.0;
  relx_err err;
  return relx_tree_attention(g_ctx, &a, 0, &err) == RELX_OK ? "ok" : err.code;
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
  say("results of any strides that are judged otherwise than by brute force", rotate_everywhere());
  say("append", append(96, 24, 8));
  say("append, head-major", append(96, 8, 32));
  say("append, pages inside slots", append(24, 48, 8));
  say("append, one page twice", append(0, 24, 8));
  say("append, slots that share elements", append(96, 20, 8));
  say("append, heads that share elements", append(96, 24, 4));
  say("attend", attend(5, 16, 2, 8));
  say("attend, one row for all", attend(5, 0, 2, 8));
  say("attend, one head for all", attend(5, 16, 2, 0));
  say("65534 blocks of heads", rotate_wide(65534, false));
  say("65536 blocks of heads", rotate_wide(65535, false));
  say("65535 blocks of heads and values", rotate_wide(43690, true));
  say("65538 blocks of heads and values", rotate_wide(43691, true));
  say("2^23 - 2 requests", attend_many((int64_t{1} << 23) - 2));
  say("2^23 - 1 requests", attend_many((int64_t{1} << 23) - 1));
  g_ctx->ctx->quarantined = true;
  say("tables of a quarantined context", tables());
  g_ctx->ctx->quarantined = false;
  if (relx_ctx_close(g_ctx, &err) != RELX_OK)
    return 1;
  fake_shutdown();
}
