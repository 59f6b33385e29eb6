// pk_strided.h - host-side checks of the ops whose matrices have row strides
// (block norm, 4-bit product, token scores): extents, overlaps, and the
// device that a call runs on.
#pragma once

#include <hip/hip_runtime.h>

#include <new>

#include "pk_abi_internal.h"

namespace pk_abi {

// `rows` rows of `row_bytes` bytes, `stride` bytes from one to the next.
struct Region {
  const void* data = nullptr;
  uint64_t rows = 0, row_bytes = 0, stride = 0;
  // Bytes from the pointer to the end of the last row.
  uint64_t extent() const { return rows ? (rows - 1) * stride + row_bytes : 0; }
};

// Whether the regions share a byte. Regions of one stride (columns of one
// buffer) and a single row, whatever stride it came with, are compared row by
// row; of two strides that interleave, any common range counts.
inline bool overlap(const Region& x, const Region& y) {
  if (!x.data || !y.data || !x.rows || !y.rows) return false;
  const uintptr_t a = reinterpret_cast<uintptr_t>(x.data), b = reinterpret_cast<uintptr_t>(y.data);
  if (a + x.extent() <= b || b + y.extent() <= a) return false;
  if (x.rows < 2 || y.rows < 2) {
    const Region &one = x.rows < 2 ? x : y, &rows = x.rows < 2 ? y : x;
    const uintptr_t p = reinterpret_cast<uintptr_t>(one.data), q = reinterpret_cast<uintptr_t>(rows.data);
    // The first of the rows that ends behind the start of the one.
    const uint64_t i = p < q + rows.row_bytes ? 0 : (p - q - rows.row_bytes) / rows.stride + 1;
    return i < rows.rows && q + i * rows.stride < p + one.row_bytes;
  }
  if (x.stride != y.stride) return true;
  const uint64_t from_x = (b >= a ? (b - a) : x.stride - (a - b) % x.stride) % x.stride;
  return from_x < x.row_bytes || x.stride - from_x < y.row_bytes;
}

// The same rows: an element of one is the element of the other.
inline bool same_rows(const Region& x, const Region& y) {
  return x.data == y.data && (x.stride == y.stride || x.rows < 2) && x.row_bytes == y.row_bytes;
}

// Makes `device` current and, at the end of the scope, the caller's again.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    status_ = hipGetDevice(&before_);
    if (status_ != hipSuccess || before_ == device) return;
    status_ = hipSetDevice(device);
    changed_ = status_ == hipSuccess;
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  hipError_t status() const { return status_; }

 private:
  int before_ = 0;
  bool changed_ = false;
  hipError_t status_ = hipSuccess;
};

// free_after_drain without changing the caller's device.
inline void free_on(int device, void* p) {
  if (!p) return;
  DeviceScope scope(device);
  (void)hipDeviceSynchronize();
  (void)hipFree(p);
}

}  // namespace pk_abi
