// fake_hip.cpp with a record of the kernels that the library has and of those that it launches, so that a test without a GPU
// sees which one a call takes.
#define hipLaunchKernel fake_launch_kernel
#include "fake_hip.cpp"
#undef hipLaunchKernel

#include <vector>

struct Launch {
    const char *name;
    unsigned grid[3];
};
static std::vector<Launch> &launched() {
    static auto *v = new std::vector<Launch>();
    return *v;
}

extern "C" {

hipError_t hipLaunchKernel(const void *f, dim3 grid, dim3 block, void **args, size_t shared, hipStream_t stream) {
    launched().push_back({names()[f].c_str(), {grid.x, grid.y, grid.z}});
    return fake_launch_kernel(f, grid, block, args, shared, stream);
}
hipError_t hipGetDevice(int *d) { return *d = 0, hipSuccess; }
hipError_t hipFuncSetAttribute(const void *, hipFuncAttribute, int) { return hipSuccess; }

void fake_forget() { launched().clear(); }
long fake_kernels() { return (long)launched().size(); }
const char *fake_kernel(long i) { return launched()[i].name; }
unsigned fake_grid(long i, int axis) { return launched()[i].grid[axis]; }
// The i-th kernel of the library, null past the last.
const char *fake_known(long i) {
    for (const auto &n : names())
        if (i-- == 0) return n.second.c_str();
    return nullptr;
}

}  // extern "C"
