// Argument checks that the C ABI layers of attention, the blocks and the 4-bit tier
// share.
#pragma once

#include "common.h"
#include "ltx25_block.h"

namespace ltx25 {

struct Rotation;
// `needed`: the tables are read; `place`: positions may be null. capi_block.cpp.
int check_rotation(const ltx25_rotation* r, bool needed, bool place, Rotation* out);

namespace checks {

// Packed tokens of a call: no sequence then has more than 2^24 units of work
// (find_unit's bound), nor 64 sequences' units more than 32 bits hold.
constexpr int kPackedMax = 1 << 27;

inline int hip_error(hipError_t e, const char* what)
{
  return set_error(LTX25_E_HIP, "%s: %s", what, hipGetErrorString(e));
}

inline bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

inline int check_aligned(const char* name, const void* p, uintptr_t align)
{
  if (!aligned(p, align)) {
    return set_error(LTX25_E_INVAL, "%s (%p) is not %d-byte aligned", name, p, (int)align);
  }
  return LTX25_OK;
}

inline int check_pointer(const char* name, const void* p, uintptr_t align)
{
  if (p == nullptr) { return set_error(LTX25_E_INVAL, "%s is null", name); }
  return check_aligned(name, p, align);
}

inline int check_tokens(const char* name, long tokens, int most)
{
  if (tokens < 0 || tokens > most) {
    return set_error(LTX25_E_INVAL, "%s=%ld is not in 0 .. %d", name, tokens, most);
  }
  return LTX25_OK;
}

inline int check_workspace(const void* workspace, size_t bytes, size_t need)
{
  const int rc = check_pointer("workspace", workspace, 16);
  if (rc == LTX25_OK && bytes < need) {
    return set_error(LTX25_E_INVAL, "the workspace has %zu bytes; this call needs %zu", bytes,
                     need);
  }
  return rc;
}

}  // namespace checks
}  // namespace ltx25
