// Buffers and uploaded matrices that outlive CloseDevice: their release must
// reach an open handle, and the handle must close once, after them.  The C
// entries that own storage are replaced by recorders here, so no GPU is used.
#include <cstdio>
#include <vector>

#include "bsp/host_code.hpp"

struct bsp_device {
  int open = 1;
  int stored = 0;
};

static int g_closed = 0, g_late = 0, g_left_at_close = 0;

extern "C" {
bsp_status bsp_device_open(int, bsp_device** out) {
  *out = new bsp_device;
  return BSP_OK;
}
bsp_status bsp_device_close(bsp_device* d) {  // the record stays readable, so that a late call shows
  g_late += !d->open;
  d->open = 0;
  g_left_at_close += d->stored;
  ++g_closed;
  return BSP_OK;
}
bsp_status bsp_buffer_alloc(bsp_device* d, int64_t bytes, void** p) {
  g_late += !d->open;
  ++d->stored;
  *p = ::operator new(static_cast<size_t>(bytes));
  return BSP_OK;
}
bsp_status bsp_buffer_free(bsp_device* d, void* p) {
  g_late += !d->open;
  --d->stored;
  ::operator delete(p);
  return BSP_OK;
}
bsp_status bsp_bsr_upload(bsp_device* d, int64_t, int64_t, int32_t, int32_t, int64_t, const int32_t*, const int32_t*,
                          const uint16_t*, bsp_bsr_desc*) {
  g_late += !d->open;
  ++d->stored;
  return BSP_OK;
}
bsp_status bsp_bsr_free(bsp_device* d, bsp_bsr_desc*) {
  g_late += !d->open;
  --d->stored;
  return BSP_OK;
}
}

int main() {
  {
    bsp::IDevice* device = bsp::CreateDevice(0);
    bsr_matrix<float> f(64, 64, 32, 32, 2, FILL_MULTI_DIAG, RAND);
    bsr_matrix<bfloat16> a = f.bfloat16_cast();
    bsp::DeviceBsr A(device, a);
    auto one = sparse_common::MakeBuffer(device, 2u, sizeof(bfloat16));
    std::shared_ptr<bsp::Buffer> other = one;
    bsp::CloseDevice(device);
  }
  {
    bsp::IDevice* device = bsp::CreateDevice(0);  // nothing stored: closes at once
    bsp::CloseDevice(device);
  }
  std::printf("closed=%d late=%d left=%d\n", g_closed, g_late, g_left_at_close);
  return !(g_closed == 2 && g_late == 0 && g_left_at_close == 0);
}
