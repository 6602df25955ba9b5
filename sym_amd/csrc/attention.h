// attention.h - arguments and launches of the paged-cache operators
// (k_tables.hip, k_rotate.hip, k_attend.h), checked and filled by
// attention.cpp. Strides are in elements unless a name says bytes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/relx.h"

#include "program.h"

namespace relx {

enum ElementType : int { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3 };

// ------------------------------------------------------------ block tables

struct TablesArgs {
  const int32_t *cached, *fresh;
  int32_t *table;
  int64_t table_row;
  const int32_t *free_pages;
  int64_t free_count;
  const int32_t *parents;
  int32_t *starts;
  int64_t *slots;
  int32_t *positions;
  int64_t *mask;
  int32_t *taken;
  FastDiv page;
  int32_t requests, columns, rows, words;
  int32_t block_rows; // rows of a block
};
hipError_t tables_launch(TablesArgs a, hipStream_t s);

// --------------------------------------------------------- norm and rotation

struct Heads {
  char *data;
  int64_t row, head;
};

struct RotateArgs {
  Heads x[3];   // queries, keys, values (values: the serving form)
  Heads y[3];   // results (serving: y[0] only); backward: the operands' gradients
  Heads dz[2];  // backward: the results' gradients
  const void *weight[2];
  const int32_t *positions;
  const float *cos, *sin;
  const int64_t *slots; // serving
  const float *scale[2];
  int64_t cache_page[2], cache_slot[2], cache_head[2];
  char *cache[2];
  float *partial; // backward: [parts, dim] per kind, queries' first
  float *weight_grad[2];
  FastDiv page;
  int64_t pages_slots; // pages * page
  int32_t weight_type;
  int32_t rows, heads[2], dim, rotary, angles, pairs;
  int32_t chunks[3]; // blocks of heads of each kind
  int32_t chunk_heads;
  float eps, inv_dim;
};
enum RotateForm : int { kRotateForward, kRotateBackward, kRotateAppend, kRotateAppendI8 };
// Blocks over the rows that a launch of `rows` rows in `chunks` blocks of
// heads takes (the backward's parts per chunk).
int rotate_blocks(int form, int64_t rows, int64_t chunks);
// Lanes that hold one head, each eight elements.
int rotate_lanes(int dim);
hipError_t rotate_launch(const RotateArgs &a, int form, int type, hipStream_t s);

// ------------------------------------------------------------ tree attention

struct AttendArgs {
  const char *q;
  int64_t q_row, q_head;
  char *out;
  int64_t out_row, out_head;
  const char *keys, *values;
  int64_t key_page, key_slot, key_head, value_page, value_slot, value_head; // bytes
  const float *key_scale, *value_scale;
  const int32_t *table;
  int64_t table_row;
  const int32_t *cached, *starts;
  const int64_t *mask;
  float *lse;
  float *partial;    // [workgroups][2][tile rows][width] sums, unnormalised
  float *stats;      // [workgroups][2][tile rows][2] maximum, sum of weights
  int64_t *schedule; // [requests + 1] first unit of each request, and their number
  FastDiv page, group;
  int32_t rows, requests, heads, kv_heads, dim, pages, columns, words;
  int32_t workgroups;
  float scale; // of a score, times log2 e
  bool once;   // in an even batch, one tile of query rows reads a key head
  // with a window (2^30: of everything) or a scale a block
  int32_t window, sinks;
  uint32_t scale_page, scale_block; // bytes
  int64_t scale_head;
  FastDiv block;
};

// How a call runs.
struct AttendPlan {
  int width;      // head size, rounded up to a kernel's
  int rows;       // query rows of an item
  bool even;      // pages of whole tiles of 16 tokens
  bool async;     // and rows of whole 16-byte pieces at 16-byte addresses
  int workgroups;
  bool quads;     // four heads of up to four rows at a time (int8 of a view)
  bool whole;     // no item is cut (a view)
};
constexpr int kMostWorkgroups = 512; // two to a compute unit

// Waves that take turns, and workgroups of them that the card holds at once: a
// ring of two tiles a wave, in 64 KiB (int8 heads of 128, say) or 128 KiB of a
// compute unit's 160. Where two fit, two: 64 requests of 512 int8 tokens at most
// with 32 key heads take 58 us with 512 workgroups, 78 with 256; up to 4096 tokens
// 248 to 258 and 246.
constexpr int turn_waves(int width) { return width == 256 ? 2 : 4; }
constexpr int turn_workgroups(int width, bool i8, bool async) {
  const int ring = 2 * 2 * 32 * width * (i8 ? 1 : 2) * turn_waves(width);
  return async ? (ring > 64 * 1024 ? kMostWorkgroups / 2 : kMostWorkgroups)
               : width == 256 ? kMostWorkgroups / 2 : kMostWorkgroups;
}
AttendPlan attend_plan(int64_t rows, int64_t requests, int64_t group, int64_t dim, int64_t page);
// Rows of partial sums that a call's workspace holds, and its bytes, whatever its
// cache's addresses.
size_t attend_part_rows(const AttendPlan &p);
size_t attend_workspace(const AttendPlan &p, int64_t requests);
hipError_t attend_launch(const AttendArgs &a, const AttendPlan &p, int type, bool i8,
                         hipStream_t s);
// The arguments of a call without a window, and how it runs; the workspace's place.
AttendArgs attend_args(const relx_tree_attention_args &p, AttendPlan &plan, int &type, bool &i8);
void attend_room(AttendArgs &a, const AttendPlan &plan, const relx_tree_attention_args &p);
hipError_t attend_launch_f16(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
hipError_t attend_launch_f16_i8(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
hipError_t attend_launch_bf16(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
hipError_t attend_launch_bf16_i8(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
// with a window; of int8 with a scale a block and a window
hipError_t attend_launch_f16_window(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
hipError_t attend_launch_f16_blocks(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
hipError_t attend_launch_bf16_window(const AttendArgs &a, const AttendPlan &p, hipStream_t s);
hipError_t attend_launch_bf16_blocks(const AttendArgs &a, const AttendPlan &p, hipStream_t s);

// ------------------------------------------------------------ blocks of a cache

struct BlockArgs {
  Heads x[2];       // keys, values
  char *cache[2];   // [pages, page, kv_heads, dim] int8
  int64_t page_stride[2], slot_stride[2], head_stride[2]; // bytes
  float *scale[2];
  int64_t scale_page, scale_block, scale_head;
  const int32_t *table;
  int64_t table_row;
  const int32_t *cached, *starts;
  FastDiv page, block;
  int32_t rows, requests, columns, pages, kv_heads, dim;
};
hipError_t blocks_launch(const BlockArgs &a, int type, hipStream_t s);

} // namespace relx
