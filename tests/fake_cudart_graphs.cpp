// Beside fake_cudart.cpp: the runtime's calls about captures and waits between streams. Loaded with it, for calls that may be captured.
#include <cuda_runtime.h>
#define EXPORT extern "C" __attribute__((visibility("default")))
static int capture = 0;
EXPORT void fake_capture(int on) { capture = on; }
EXPORT cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* s) {
  *s = capture ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
EXPORT cudaError_t cudaStreamWaitEvent(cudaStream_t, cudaEvent_t, unsigned) { return cudaSuccess; }
