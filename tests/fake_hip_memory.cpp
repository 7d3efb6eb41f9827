// The stand-in runtime of fake_hip.cpp that also watches memory: which allocations there are, and whether a copy from the host changes one that
// a launch before it may still read.  A launch counts as under way until something waits for the device: hipDeviceSynchronize, or
// hipFree of memory.  (hipMemcpy waits for the default stream alone, not for streams that were made non-blocking.)
//
// Log lines besides fake_hip.cpp's:  malloc <address> <bytes> | unordered <address> <bytes>
#define hipMalloc plain_hipMalloc
#define hipFree plain_hipFree
#define hipMemcpy plain_hipMemcpy
#define hipLaunchKernel plain_hipLaunchKernel
#define hipGetDevice plain_hipGetDevice
#include "fake_hip.cpp"
#undef hipMalloc
#undef hipFree
#undef hipMemcpy
#undef hipLaunchKernel
#undef hipGetDevice

namespace {

std::map<char*, size_t>& allocations() {
    static std::map<char*, size_t> m;
    return m;
}
std::set<char*>& being_read() {  // by launches under way: all that was there when they were launched
    static std::set<char*> s;
    return s;
}
long copies = 0, fail_copy = -1;
int device = 0;

}  // namespace

extern "C" {

void fake_fail_copy(long which) { fail_copy = which < 0 ? -1 : copies + which; }  // counted from the next one; none from a negative number on
void fake_set_device(int d) { device = d; }

hipError_t hipMalloc(void** p, size_t n) {
    const hipError_t e = plain_hipMalloc(p, n);
    if (e != hipSuccess) return e;
    Own own;
    allocations()[static_cast<char*>(*p)] = n;
    note("malloc", std::to_string(reinterpret_cast<unsigned long long>(*p)).c_str(), (int)n);
    return e;
}
hipError_t hipDeviceSynchronize() {
    being_read().clear();
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (p) {
        Own own;
        being_read().clear();
        allocations().erase(static_cast<char*>(p));
    }
    return plain_hipFree(p);
}
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind kind) {
    if (copies++ == fail_copy) return report(hipErrorUnknown);
    Own own;
    for (char* a : being_read())
        if (static_cast<char*>(d) < a + allocations()[a] && a < static_cast<char*>(d) + n)
            note("unordered", std::to_string(reinterpret_cast<unsigned long long>(d)).c_str(), (int)n);
    return plain_hipMemcpy(d, s, n, kind);
}
hipError_t hipLaunchKernel(const void* f, dim3 grid, dim3 block, void** args, size_t lds, hipStream_t s) {
    {
        Own own;
        for (auto& a : allocations()) being_read().insert(a.first);
    }
    return plain_hipLaunchKernel(f, grid, block, args, lds, s);
}
hipError_t hipGetDevice(int* d) {
    *d = device;
    return hipSuccess;
}

}  // extern "C"
