// capi.h - what the C entry points (capi.cpp, attention.cpp) share: the
// context handle and the boundary that no exception crosses.
#pragma once

#include <cstdio>
#include <cstring>
#include <memory>
#include <new>
#include <string>

#include "../../include/relx.h"
#include "plan.h"

namespace relx {
struct Context;
}

struct relx_ctx {
  std::shared_ptr<relx::Context> ctx;
};

namespace {

inline void set_err(relx_err *err, const std::string &code, const std::string &msg,
                    int64_t offset = -1, int completion = RELX_NOT_LAUNCHED) {
  if (!err)
    return;
  std::memset(err, 0, sizeof(*err));
  std::snprintf(err->code, sizeof(err->code), "%s", code.c_str());
  std::snprintf(err->message, sizeof(err->message), "%s", msg.c_str());
  err->offset = offset;
  err->completion = completion;
}

inline void clear_err(relx_err *err) {
  if (err) {
    std::memset(err, 0, sizeof(*err));
    err->offset = -1;
  }
}

template <class F> int guarded(relx_err *err, F &&fn) {
  try {
    clear_err(err);
    fn();
    return RELX_OK;
  } catch (const relx::Error &e) {
    set_err(err, e.code, e.message, e.offset);
  } catch (const std::bad_alloc &) {
    set_err(err, "out_of_memory", "host allocation failed");
  } catch (const std::exception &e) {
    set_err(err, "internal_error", e.what());
  }
  return RELX_ERROR;
}

} // namespace
