// Status and error plumbing of the C ABI, needed by every other source.
#include "common.cuh"

#include <cstdlib>

namespace b200q {

static thread_local int g_last_cuda = 0;
int status_from(cudaError_t e) {
    if (e == cudaSuccess) return B200Q_OK;
    g_last_cuda = (int)e;
    return B200Q_ECUDA;
}
bool pdl_enabled() {
    static const bool on = [] { const char* e = getenv("B200Q_PDL"); return !(e && atoi(e) == 0); }();
    return on;
}

int device_sms() {
    static int sms[64] = {0};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64) dev = 0;
    if (!sms[dev]) {
        int v = 0;
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
        sms[dev] = v > 0 ? v : 148;
    }
    return sms[dev];
}

// the error words of the sources that keep one, weak: a library built without the IQ2_XXS tables leaves two of them out
__attribute__((weak)) int iq2_error_read(int clear);    // iq2.cu
__attribute__((weak)) int tc_error_read(int clear);     // tc_gemm.cu
__attribute__((weak)) int nv4_error_read(int clear);    // nv4_gemm.cu
__attribute__((weak)) int gemv_error_read(int clear);   // gemv_tc.cu
__attribute__((weak)) int kv_error_read(int clear);     // kv.cu
__attribute__((weak)) int attn_error_read(int clear);   // attn_decode.cu
__attribute__((weak)) int prompt_error_read(int clear); // attn_prompt.cu

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_abi(void) { return B200Q_ABI; }
int b200q_last_cuda_error(void) { return g_last_cuda; }
const char* b200q_strerror(int status) {
    switch (status) {
        case B200Q_OK: return "ok";
        case B200Q_EINVAL: return "invalid argument (null pointer, shape or alignment)";
        case B200Q_ENOSPACE: return "workspace or capacity too small";
        case B200Q_ECUDA: return "CUDA launch error (see b200q_last_cuda_error)";
        default: return "unknown status";
    }
}

int b200q_device_error(int clear) {
    const struct { int (*read)(int); int shift; } words[] = {
        {iq2_error_read, 0}, {tc_error_read, 4}, {nv4_error_read, 8}, {gemv_error_read, 12}, {kv_error_read, 16},
        {attn_error_read, 20}, {prompt_error_read, 20}};   // both forms of the paged attention report alike
    int v = 0;
    for (const auto& w : words) {
        const int e = w.read ? w.read(clear) : 0;
        if (e < 0) return -1;
        v |= e << w.shift;
    }
    return v;
}

}  // extern "C"
