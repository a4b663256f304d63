// Stands in for the HIP runtime where the kernel library is loaded without a GPU: launches are written down, not made.
#include <cstddef>
#include <cstdint>
#include <string>
#include <unordered_map>

namespace {
struct Dim {
  uint32_t x, y, z;
};
std::unordered_map<const void*, std::string>& names() {
  static auto* all = new std::unordered_map<const void*, std::string>;
  return *all;
}
std::string made;
Dim grid, block;
size_t lds;
void* queue;
}  // namespace

extern "C" {
void** __hipRegisterFatBinary(const void*) {
  static void* none = nullptr;
  return &none;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterVar(void**, void*, char*, char*, int, size_t, int, int) {}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*) {
  names()[host] = name;
}
int __hipPushCallConfiguration(Dim g, Dim b, size_t shared, void* stream) {
  grid = g, block = b, lds = shared, queue = stream;
  return 0;
}
int __hipPopCallConfiguration(Dim* g, Dim* b, size_t* shared, void** stream) {
  *g = grid, *b = block, *shared = lds, *stream = queue;
  return 0;
}
int hipLaunchKernel(const void* kernel, Dim g, Dim b, void**, size_t shared, void*) {
  made += names()[kernel] + " " + std::to_string(g.x) + " " + std::to_string(b.x) + " " + std::to_string(shared) + "\n";
  return 0;
}
int hipGetLastError() { return 0; }
int hipFuncSetAttribute(const void*, int, int) { return 0; }

// What was launched since the last call: a line each of the kernel's name, workgroups, threads, bytes of LDS asked for.
const char* launches() {
  static std::string last;
  last.swap(made);
  made.clear();
  return last.c_str();
}
// The names of all kernels.
const char* kernels() {
  static std::string all;
  all.clear();
  for (const auto& k : names()) all += k.second + "\n";
  return all.c_str();
}
}
