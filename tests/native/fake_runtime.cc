// A stand-in for the few CUDA runtime calls that the host checks reach (cudaError_t
// is an int to the linker). `fake_last` is what the runtime remembers.
extern "C" {
int fake_last = 0;

int cudaGetLastError() {
    const int e = fake_last;
    fake_last = 0;
    return e;
}
int cudaPeekAtLastError() { return fake_last; }
const char *cudaGetErrorName(int) { return "name"; }
const char *cudaGetErrorString(int) { return "text"; }
int cudaGetDevice(int *dev) { return *dev = 0; }
int cudaDeviceGetAttribute(int *value, int, int) {
    *value = 148;
    return 0;
}

// what nvcc's start-up code calls: there is no device code to register here
void **__cudaRegisterFatBinary(void *) { return nullptr; }
void __cudaRegisterFatBinaryEnd(void **) {}
void __cudaUnregisterFatBinary(void **) {}
char __cudaInitModule(void **) { return 0; }
}
