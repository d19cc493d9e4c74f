// The stream kernel of window_stream.h over e2m1 caches.
#include "window_stream.h"

int dsp_window::stream_fp4(int32_t D, int32_t dtype, const WinPlan& p, const WinArgs& a,
                           hipStream_t s) {
  return stream_format<kFp4>(D, dtype, p, a, s);
}
