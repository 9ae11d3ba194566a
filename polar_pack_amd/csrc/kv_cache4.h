// Appending to and reading from the 4-bit cache (kv_cache4.hip).
#pragma once

#include "kv_append.h"
#include "rotary.h"

namespace pp {

struct ReadArgs {
  KvCache C;
  KvSeqs S;
  void* out[2];
};

// `rot` null: keys as they are, no queries; otherwise keys turned, and the queries' rows too.
int kv_append4(const AppendArgs& A, const Rot* rot, const RotRows* q, int D, int dtype, hipStream_t st);
int kv_read4(const ReadArgs& A, int D, int dtype, hipStream_t st);

}  // namespace pp
