// C ABI of eii_sample: argument checks, handle, launch.
#include <cuda_runtime.h>

#include <cstdint>
#include <new>

#include "eii.h"
#include "eii_host.h"
#include "eii_sample.cuh"

using namespace eii;

struct eii_sampler {
    int device = 0, num_sms = 0;
    int* err = nullptr;
};

namespace {

int launch_sample(const eii_sampler* s, const SampleParams& p, int cs, cudaStream_t st) {
    const int rows_at_once = s->num_sms / cs > 0 ? s->num_sms / cs : 1;
    const int ch = (p.vocab + cs * 4 * SAMPLE_THREADS - 1) / (cs * 4 * SAMPLE_THREADS);
    const int aligned = ((reinterpret_cast<uintptr_t>(p.logits) | static_cast<uintptr_t>(p.ld * 4)) & 15) == 0;
    cudaLaunchConfig_t cfg{};
    cfg.stream = st;
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.gridDim = dim3(static_cast<unsigned>(cs * (p.n_rows < rows_at_once ? p.n_rows : rows_at_once)));
    cfg.dynamicSmemBytes = ch * 16 * SAMPLE_THREADS + sizeof(SampleShared);
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cs;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    CK(cudaLaunchKernelEx(&cfg, k_sample, p, cs, ch, aligned));
    return EII_OK;
}

// Once per handle: the kernel's shared memory on the current device.
int allow_sample() {
    CK(cudaFuncSetAttribute(k_sample, cudaFuncAttributeMaxDynamicSharedMemorySize,
                            SAMPLE_MAX_CHUNKS * 16 * SAMPLE_THREADS + static_cast<int>(sizeof(SampleShared))));
    return EII_OK;
}

}  // namespace

extern "C" {

int eii_sampler_open(int device, eii_sampler** out) {
    if (!out) return fail(EII_ERR_ARG, "out is null");
    *out = nullptr;
    TRY(check_device(device));
    DeviceGuard dg(device);
    CK(dg.st);
    eii_sampler* s = new (std::nothrow) eii_sampler;
    if (!s) return fail(EII_ERR_ARG, "out of host memory");
    s->device = device;
    if (cudaDeviceGetAttribute(&s->num_sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
        cudaMalloc(&s->err, 16) != cudaSuccess || cudaMemset(s->err, 0, 16) != cudaSuccess ||
        cudaStreamSynchronize(nullptr) != cudaSuccess) {  // (a memset may return before it is done)
        const int rc = fail(EII_ERR_CUDA, "sampler set-up failed: %s", cudaGetErrorString(cudaGetLastError()));
        cudaFree(s->err);
        delete s;
        return rc;
    }
    const int rc = allow_sample();
    if (rc != EII_OK) {
        cudaFree(s->err);
        delete s;
        return rc;
    }
    *out = s;
    return EII_OK;
}

int eii_sample(eii_sampler* s, const int32_t* logits, int64_t ld, int n_rows, int vocab, const int32_t* inv_temp,
               const int32_t* top_k, const int32_t* top_p, const int32_t* min_p, const uint32_t* u, int64_t* token,
               int32_t* kept, int32_t* prob, void* stream) {
    if (!s) return fail(EII_ERR_ARG, "sampler is null");
    // (a block's next row, the grid's width further on, has to be an int)
    if (n_rows < 0 || n_rows > SAMPLE_MAX_ROWS) return fail(EII_ERR_ARG, "n_rows must be in [0, %d] (got %d)", SAMPLE_MAX_ROWS, n_rows);
    if (n_rows == 0) return EII_OK;
    if (!logits || !u || !token) return fail(EII_ERR_ARG, "logits, u or token is null");
    if (vocab < 1 || vocab > SAMPLE_MAX_VOCAB) return fail(EII_ERR_ARG, "vocab must be in [1, %d] (got %d)", SAMPLE_MAX_VOCAB, vocab);
    if (ld < vocab) return fail(EII_ERR_ARG, "ld must be >= %d (got %lld)", vocab, (long long)ld);
    const struct { const char* name; const void* p; } words[] = {{"logits", logits}, {"u", u}, {"inv_temp", inv_temp}, {"top_k", top_k},
                                                                 {"top_p", top_p}, {"min_p", min_p}, {"kept", kept}, {"prob", prob}};
    for (const auto& w : words) TRY(check_aligned(w.name, w.p, 4));
    TRY(check_aligned("token", token, 8));
    DeviceGuard dg(s->device);
    CK(dg.st);
    SampleParams p{};
    p.logits = logits; p.ld = ld; p.n_rows = n_rows; p.vocab = vocab; p.inv_temp = inv_temp; p.top_k = top_k;
    p.top_p = top_p; p.min_p = min_p; p.u = u; p.token = token; p.kept = kept; p.prob = prob; p.err = s->err;
    // Blocks per row: as many as its weights need, and up to four while that leaves no row waiting (one row of
    // 49152: 38 us on one block, 24 on two, 20 on four, 21 on eight).
    int cs = 1;
    while (cs * SAMPLE_MAX_CHUNKS * 4 * SAMPLE_THREADS < vocab || (cs < 4 && n_rows <= s->num_sms / (2 * cs) && cs * 4 * SAMPLE_THREADS < vocab))
        cs *= 2;
    return launch_sample(s, p, cs, static_cast<cudaStream_t>(stream));
}

int eii_sampler_sync(eii_sampler* s, void* stream) {
    if (!s) return fail(EII_ERR_ARG, "sampler is null");
    DeviceGuard dg(s->device);
    CK(dg.st);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int code = 0;
    CK(cudaMemcpyAsync(&code, s->err, sizeof(int), cudaMemcpyDeviceToHost, st));
    CK(cudaStreamSynchronize(st));
    if (!code) return EII_OK;
    CK(cudaMemsetAsync(s->err, 0, sizeof(int), st));
    CK(cudaStreamSynchronize(st));
    if (code == ERR_SAMPLE_PARAM) return fail(EII_ERR_ARG, "a row's sampling parameter lies outside its range");
    return fail(EII_ERR_DEVICE, "kernel reported error %d", code);
}

void eii_sampler_close(eii_sampler* s) {
    if (!s) return;
    DeviceGuard dg(s->device);
    cudaFree(s->err);
    delete s;
}

}  // extern "C"
