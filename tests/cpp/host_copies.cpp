// The copies of llmc_b200.hpp are ordered with a context's work.  Runs on the CPU: the CUDA runtime and the library's
// entry points are stand-ins over host memory with two queues that do not wait for one another, as a non-blocking
// stream and the legacy stream do not.  With `late` a context's work runs only when something waits for it (a read
// that did not wait finds the old values); without, it runs at once (an upload that was not waited for is not there).
// A copy to the device or on it is queued when cudaMemcpy returns, a copy to the host is made in it.
#include <cstdio>
#include <cstdlib>

#include "llmc_b200.hpp"

namespace {
bool late = false;
std::vector<std::function<void()>> own, legacy;
int failed = 0;

void drain(std::vector<std::function<void()>>& q) {
    for (auto& f : q) f();
    q.clear();
}
llmc_status launch(std::function<void()> f) {
    own.push_back(std::move(f));
    if (!late) drain(own);
    return LLMC_OK;
}
void expect(const char* what, double got, double want) {
    if (got == want) return;
    std::printf("FAIL %s (work %s): got %g, want %g\n", what, late ? "late" : "early", got, want);
    failed++;
}
}  // namespace

// ---- the CUDA runtime --------------------------------------------------------------------------
extern "C" {
cudaError_t cudaGetDevice(int* d) { return *d = 0, cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "error"; }
cudaError_t cudaMalloc(void** p, size_t n) { return *p = std::calloc(1, n), cudaSuccess; }
cudaError_t cudaFree(void* p) {  // waits for the device, as the runtime's does
    drain(legacy);
    drain(own);
    std::free(p);
    return cudaSuccess;
}
cudaError_t cudaMemcpy(void* dst, const void* src, size_t n, cudaMemcpyKind kind) {
    if (kind == cudaMemcpyDeviceToHost) {
        drain(legacy);
        std::memcpy(dst, src, n);
    } else if (kind == cudaMemcpyHostToDevice) {
        std::vector<unsigned char> staged((const unsigned char*)src, (const unsigned char*)src + n);
        legacy.push_back([=] { std::memcpy(dst, staged.data(), n); });
    } else {
        legacy.push_back([=] { std::memcpy(dst, src, n); });
    }
    return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() {
    drain(legacy);
    drain(own);
    return cudaSuccess;
}
cudaError_t cudaStreamSynchronize(cudaStream_t s) {
    drain(s == cudaStreamLegacy ? legacy : own);
    return cudaSuccess;
}

// ---- the library: what the tests call, over flat arrays ------------------------------------------
const char* llmc_last_error(void) { return ""; }
llmc_status llmc_init(int32_t, llmc_ctx** out) { return *out = (llmc_ctx*)&late, LLMC_OK; }
llmc_status llmc_destroy(llmc_ctx*) { return LLMC_OK; }
llmc_status llmc_chol_inverse(llmc_ctx*, const float* H, int64_t d, int64_t, float, int32_t, float* out, int64_t, int32_t) {
    return launch([=] {
        for (int64_t i = 0; i < d * d; i++) out[i] = i % (d + 1) ? 0.f : 1.f / H[i];
    });
}
llmc_status llmc_observer_minmax(llmc_ctx*, const void* x, int32_t, int64_t rows, int64_t cols, int64_t, int32_t, int64_t, float* mn, float* mx,
                                 int32_t) {
    return launch([=] {
        for (int64_t i = 0; i < rows * cols; i++) {
            const float v = ((const float*)x)[i];
            if (v < *mn) *mn = v;
            if (v > *mx) *mx = v;
        }
    });
}
llmc_status llmc_affine_params(llmc_ctx*, const float* mn, const float* mx, int64_t n, int32_t, int32_t, float* s, int32_t* z) {
    return launch([=] {
        for (int64_t i = 0; i < n; i++) {
            s[i] = mx[i] - mn[i];
            z[i] = (int32_t)mn[i];
        }
    });
}
llmc_status llmc_fake_quantize(llmc_ctx*, const void* x, int32_t, int64_t n, float s, int32_t, int32_t, int32_t, void* out, int32_t* codes) {
    return launch([=] {
        for (int64_t i = 0; i < n; i++) {
            if (out) ((float*)out)[i] = ((const float*)x)[i] + s;
            if (codes) codes[i] = (int32_t)((const float*)x)[i];
        }
    });
}
llmc_status llmc_int4_pack(llmc_ctx*, const int32_t* codes, int64_t n, int32_t, uint8_t* out) {
    return launch([=] {
        for (int64_t i = 0; i + 1 < n; i += 2) out[i / 2] = (uint8_t)(codes[i] * 16 + codes[i + 1]);
    });
}
llmc_status llmc_int4_unpack_dequant(llmc_ctx*, const uint8_t* in, int64_t n, float s, int32_t, int32_t, float* out) {
    return launch([=] {
        for (int64_t i = 0; i < n; i++) out[i] = s * (i % 2 ? in[i / 2] & 15 : in[i / 2] >> 4);
    });
}
llmc_status llmc_observer_mse(llmc_ctx*, const void* x, int32_t, int64_t n, int32_t, int32_t, int32_t, float* s, int32_t* z, double*) {
    own.push_back([=] {  // waits for its stream itself: it returns host values
        *s = 0;
        for (int64_t i = 0; i < n; i++) *s += ((const float*)x)[i];
        *z = 0;
    });
    drain(own);
    return LLMC_OK;
}
llmc_status llmc_rtn_quantize(llmc_ctx*, const void* w, int32_t, int64_t m, int64_t n, int64_t, const llmc_qconfig*, uint8_t* codes, float* s,
                              int32_t* z, void* deq) {
    return launch([=] {
        for (int64_t i = 0; i < m * ((n + 1) / 2); i++) codes[i] = 7;
        for (int64_t i = 0; i < m; i++) {
            s[i] = ((const float*)w)[i * n];
            z[i] = 3;
        }
        for (int64_t i = 0; i < m * n; i++) ((float*)deq)[i] = ((const float*)w)[i];
    });
}
}  // extern "C"

int main() {
    using namespace llmcs;
    for (bool l : {true, false}) {
        late = l;
        Context c;
        {  // an upload, a solve and its read-back
            const auto h = HessianInverseSolver::Compute(c, DeviceTensor::FromHost({2, 0, 0, 2}, {2, 2}), 0.f).ToHost();
            expect("Compute", h[0], 0.5);
        }
        {  // the observer's first values and its parameters
            MinMaxObserver o(c);
            const DeviceTensor x = DeviceTensor::FromHost({-3, 5}, {1, 2});
            o.Update(x);
            const QuantizationParameters p = o.GetQuantParams(4, false);
            expect("MinMaxObserver scale", p.Scale[0], 8);
            expect("MinMaxObserver zero", (double)p.ZeroPoint[0], -3);
        }
        {  // copies of what a context's work has made, and their joining
            MSEObserver o(c);
            const DeviceTensor x = DeviceTensor::FromHost({1, 2}, {2});
            const DeviceTensor y = FakeQuantize::Apply(c, x, 10.f, 0, 4, true);
            o.Update(y);
            expect("MSEObserver, one batch", o.GetQuantParams(4, true).Scale[0], 23);
            o.Update(x);
            expect("MSEObserver, two batches", o.GetQuantParams(4, true).Scale[0], 26);
        }
        {
            const DeviceTensor x = DeviceTensor::FromHost({1, 2, 3, 4}, {4});
            const Int4PackedTensor t = Int4PackedTensor::FromFloat(c, x, 1.f, 0, true);
            expect("Int4PackedTensor", t.PackedBytes()[1], 0x34);
            expect("Int4PackedTensor, from bytes", Int4PackedTensor::FromPackedBytes(c, {0x12, 0x34}, 4, 2.f, 0, true).Dequantize().ToHost()[3], 8);
        }
        {  // raw bytes
            const RtnResult r = Rtn::Quantize(c, DeviceTensor::FromHost({6, 1}, {1, 2}), RtnConfig{});
            expect("Rtn codes", r.Codes[0], 7);
            expect("Rtn scale", r.Scales[0], 6);
            expect("Rtn zero", r.ZeroPoints[0], 3);
            expect("Rtn weight", r.Dequantized.ToHost()[0], 6);
        }
    }
    std::printf("%d failed\n", failed);
    return failed != 0;
}
