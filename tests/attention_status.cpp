// The self-check word of cross attention against a CUDA runtime made up here: one word of a "device" that is host memory, copies that run
// at once, and a kernel that fails at a chosen moment.  cross_attention.cu is compiled into this file.
//
// Usage: attention_status SCENARIO; exits with 0 if it holds, else prints what does not.
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>

#include "cross_attention.cu"

namespace {

std::string last_error;
std::function<void()> after_copy = [] {};
int failures = 0;

void check(bool holds, const char* what, int line) {
  if (!holds) {
    std::printf("line %d: %s (%s)\n", line, what, last_error.c_str());
    failures++;
  }
}
#define CHECK(x) check((x), #x, __LINE__)

}  // namespace

namespace mlxd {
int fail(int code, const std::string& msg) {
  last_error = msg;
  return code;
}
int fail_cuda(cudaError_t, const char* what) { return fail(MLXD_ERR_CUDA, what); }
int device_sms(int, int* sms) {
  *sms = 148;
  return MLXD_OK;
}
bool takes_steps(const CrossParams&, int) { return false; }
size_t step_workspace(const CrossParams&, int) { return 0; }
cudaError_t launch_cross_step(const CrossParams&, void*, int, int, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t launch_cross_forward(const CrossParams&, const CrossMaps&, int, cudaStream_t) { return cudaErrorNotSupported; }
cudaError_t launch_cross_backward(const CrossParams&, const CrossMaps&, int, cudaStream_t) { return cudaErrorNotSupported; }
}  // namespace mlxd

extern "C" {
cudaError_t cudaGetDevice(int* d) {
  *d = 0;
  return cudaSuccess;
}
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetSymbolAddress(void** at, const void* symbol) {
  *at = const_cast<void*>(symbol);
  return cudaSuccess;
}
cudaError_t cudaMemcpyAsync(void* d, const void* s, size_t n, cudaMemcpyKind, cudaStream_t) {
  std::memcpy(d, s, n);
  after_copy();
  return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void* d, int v, size_t n, cudaStream_t) {
  std::memset(d, v, n);
  return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t) { return cudaSuccess; }
cudaError_t cudaGetDriverEntryPoint(const char*, void**, unsigned long long, cudaDriverEntryPointQueryResult*) { return cudaErrorNotSupported; }
}

namespace {

cudaStream_t stream(int i) { return reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(16 * i)); }

int ask(int of, int32_t* word) { return mlxd_attention_status(0, stream(of), word); }

// Whoever asks learns of a failure, also after another stream's owner has asked.
void two_askers() {
  int32_t word = -1;
  CHECK(ask(1, &word) == MLXD_OK && word == 0);
  attention_status = 1;
  CHECK(ask(1, &word) == MLXD_ERR_DEVICE && word == 1);
  CHECK(ask(2, &word) == MLXD_ERR_DEVICE && word == 1);
}

// A kernel on another stream fails while the word is being read.
void failure_while_asking() {
  int32_t word = -1;
  after_copy = [] { attention_status = 1; };
  CHECK(ask(1, &word) == MLXD_OK && word == 0);
  after_copy = [] {};
  CHECK(ask(1, &word) == MLXD_ERR_DEVICE && word == 1);
}

}  // namespace

int main(int argc, char** argv) {
  const std::string scenario = argc > 1 ? argv[1] : "";
  if (scenario == "two_askers") two_askers();
  else if (scenario == "failure_while_asking") failure_while_asking();
  else return 2;
  return failures ? 1 : 0;
}
