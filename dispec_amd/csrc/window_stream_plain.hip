// The stream kernel of window_stream.h over caches in the model's type.
#include "window_stream.h"

int dsp_window::stream_plain(int32_t D, int32_t dtype, const WinPlan& p, const WinArgs& a,
                           hipStream_t s) {
  return stream_format<kNone>(D, dtype, p, a, s);
}
