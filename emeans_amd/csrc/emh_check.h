// What the learning operators' entry points check before anything is queued, and how
// they report it (emh_learn.cpp, emh_answer.cpp).
#pragma once

#include <exception>

#include "emh_learn.h"

namespace {

template <class F>
int guard(F&& f) {
  try {
    f();
    return EMH_OK;
  } catch (const emh::Invalid& e) {
    emh::set_last_error(e.what());
    return EMH_INVALID;
  } catch (const std::exception& e) {
    emh::set_last_error(e.what());
    return EMH_ERROR;
  } catch (...) {
    emh::set_last_error("unknown error");
    return EMH_ERROR;
  }
}

void use_device(emh_ctx* c) { EMH_HIP(hipSetDevice(c->device)); }

bool real_kind(int k) { return k == EMH_F32 || k == EMH_F16 || k == EMH_BF16; }

// The bytes that an operand covers.
struct Range {
  const char* lo = nullptr;
  const char* hi = nullptr;
  bool meets(const Range& o) const { return lo < o.hi && o.lo < hi; }
  bool same(const Range& o) const { return lo == o.lo && hi == o.hi; }
};
Range range_of(const void* p, size_t len, int kind) {
  return {(const char*)p, (const char*)p + len * emh::kind_bytes(kind)};
}

void check_address(const emh_buf* b, const char* what) {
  EMH_ENSURE((uintptr_t)b->ptr % emh::kind_bytes(b->kind) == 0,
             "%s does not begin at an element's address", what);
}

// A rows x d matrix with row stride ld (0: d) in b; its stride and range.
Range check_matrix(const emh_buf* b, size_t rows, size_t d, size_t& ld, const char* what) {
  if (ld == 0) ld = d;
  EMH_ENSURE(ld >= d, "%s: the row stride %zu is less than the row's %zu", what, ld, d);
  check_address(b, what);
  size_t span = 0;
  if (rows > 0)
    EMH_ENSURE(!__builtin_mul_overflow(rows - 1, ld, &span) &&
                   !__builtin_add_overflow(span, d, &span) && span <= b->len,
               "%s: the buffer's %zu elements do not hold %zu rows of %zu (stride %zu)", what,
               b->len, rows, d, ld);
  return range_of(b->ptr, span, b->kind);
}
Range check_vector(const emh_buf* b, size_t len, const char* what) {
  EMH_ENSURE(b->len >= len, "%s: the buffer's %zu elements are fewer than %zu", what, b->len, len);
  check_address(b, what);
  return range_of(b->ptr, len, b->kind);
}
Range check_f32(const emh_buf* b, size_t len, const char* what) {
  EMH_ENSURE(b && b->kind == EMH_F32, "%s must be an f32 buffer", what);
  return check_vector(b, len, what);
}
void apart(const Range& out, const Range& in, const char* a, const char* b) {
  EMH_ENSURE(!out.meets(in), "%s overlaps %s", a, b);
}
void apart_or_same(const Range& out, const Range& in, bool same_ld, const char* a, const char* b) {
  EMH_ENSURE(!out.meets(in) || (out.same(in) && same_ld), "%s overlaps %s in part", a, b);
}
constexpr size_t MAX_D = size_t(1) << 30;

// A norm's weight or bias: d entries of x's kind or f32.
emh::MatIn check_affine(const emh_buf* b, size_t d, int kind, const char* what, Range& r) {
  if (!b) return {};
  EMH_ENSURE(b->kind == EMH_F32 || b->kind == kind, "%s must be f32 or of x's kind", what);
  r = check_vector(b, d, what);
  return {b->ptr, d, b->kind};
}

}  // namespace
