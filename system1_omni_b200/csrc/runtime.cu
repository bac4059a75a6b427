// The CUDA runtime calls a caller of libqwen3_5_cuda.so needs, so that a host that loads
// this one library never links CUDA itself (reference: src/backends/cuda/qwen3_5/runtime.cu:9-74).
#include <cuda_runtime.h>

#include "common.cuh"
#include "cs1_ops.h"
#include "s1_executor.h"

extern "C" {

uint32_t cs1_abi_version(void) { return CS1_ABI_VERSION; }

// A static string for any code: CUDA's for cudaError_t values, this library's above 1000.
const char* cs1_error_string(int code) {
    if (code >= CS1_ERR_GEMM_BASE && code < CS1_ERR_UNSUPPORTED) return "GEMM handle or engine error (code - 1000)";
    switch (code) {
        case CS1_ERR_UNSUPPORTED: return "operation not built into this library";
        case CS1_ERR_DEVICE_CHECK: return "a device-side bounded wait gave up";
        case CS1_ERR_TENSOR_MAP: return "TMA tensor map encoding failed";
        case CS1_ERR_STATIC_SCRATCH: return "window larger than the fixed scratch of cs1_gdn_prefill_static";
        case 3000: return "executor: invalid argument";
        case 3001: return "executor: a logit is not finite";
        case 3002: return "executor: no tensor of that name in the decoder";
        case 3003: return "executor: tensor size differs from the planned one";
        case 3004: return "checkpoint: file cannot be opened or mapped";
        case 3005: return "checkpoint: not a safetensors file or index";
        case 3006: return "checkpoint: tensor is not bfloat16";
        case 3007: return "checkpoint: embed_tokens.weight or a tensor of the decoder is missing";
        case 3008: return "export manifest: a field is missing or invalid";
        case 3009: return "pages: not enough free pages, table room or list room";
        case 3100: return "dispatcher: libnccl.so.2 cannot be loaded";
        case 3101: return "dispatcher: the communicator id could not be exchanged";
        case 3102: return "dispatcher: an NCCL call failed";
        case 3103: return "dispatcher: call out of order";
        default: break;
    }
    return cudaGetErrorString(static_cast<cudaError_t>(code));
}

int cs1_set_device(int device) { return cudaSetDevice(device); }
int cs1_malloc(void** ptr, size_t bytes) { return cudaMalloc(ptr, bytes); }
int cs1_free(void* ptr) { return cudaFree(ptr); }

int cs1_stream_create(void** stream) {
    return cudaStreamCreateWithFlags(reinterpret_cast<cudaStream_t*>(stream), cudaStreamNonBlocking);
}
int cs1_stream_destroy(void* stream) { return cudaStreamDestroy(static_cast<cudaStream_t>(stream)); }
int cs1_stream_sync(void* stream) { return cudaStreamSynchronize(static_cast<cudaStream_t>(stream)); }

int cs1_upload(void* dst, const void* src, size_t bytes, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cudaMemcpyAsync(dst, src, bytes, cudaMemcpyHostToDevice, st);
    return e != cudaSuccess ? e : cudaStreamSynchronize(st);
}

int cs1_download(void* dst, const void* src, size_t bytes, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToHost, st);
    return e != cudaSuccess ? e : cudaStreamSynchronize(st);
}

int cs1_copy_dd(void* dst, const void* src, size_t bytes, void* stream) {
    const cudaError_t e =
        cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToDevice, static_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? e : cudaGetLastError();
}

int cs1_copy2d(void* dst, size_t dpitch, const void* src, size_t spitch, size_t width, size_t height,
               void* stream) {
    const cudaError_t e = cudaMemcpy2DAsync(dst, dpitch, src, spitch, width, height, cudaMemcpyDeviceToDevice,
                                            static_cast<cudaStream_t>(stream));
    return e != cudaSuccess ? e : cudaGetLastError();
}

// Thread-local capture so that other threads' CUDA calls do not invalidate it; a failed
// begin/end clears the sticky error so the next capture can start (runtime.cu:52-66).
int cs1_graph_begin(void* stream) {
    const cudaError_t e = cudaStreamBeginCapture(static_cast<cudaStream_t>(stream), cudaStreamCaptureModeThreadLocal);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e;
}

int cs1_graph_end(void* stream, void** exec) {
    cudaGraph_t graph = nullptr;
    cudaError_t e = cudaStreamEndCapture(static_cast<cudaStream_t>(stream), &graph);
    if (e == cudaSuccess) e = cudaGraphInstantiate(reinterpret_cast<cudaGraphExec_t*>(exec), graph, 0);
    if (graph) cudaGraphDestroy(graph);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e;
}

int cs1_graph_launch(void* exec, void* stream) {
    const cudaError_t e = cudaGraphLaunch(static_cast<cudaGraphExec_t>(exec), static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e;
}

int cs1_graph_destroy(void* exec) { return cudaGraphExecDestroy(static_cast<cudaGraphExec_t>(exec)); }

// ---- additions for hosts that also time and stage through this library ----

int s1_device_count(int* count) { return cudaGetDeviceCount(count); }
int s1_event_create(void** event) { return cudaEventCreate(reinterpret_cast<cudaEvent_t*>(event)); }
int s1_event_destroy(void* event) { return cudaEventDestroy(static_cast<cudaEvent_t>(event)); }
int s1_event_record(void* event, void* stream) {
    return cudaEventRecord(static_cast<cudaEvent_t>(event), static_cast<cudaStream_t>(stream));
}
int s1_event_sync(void* event) { return cudaEventSynchronize(static_cast<cudaEvent_t>(event)); }
int s1_event_elapsed_ms(void* start, void* stop, float* ms) {
    return cudaEventElapsedTime(ms, static_cast<cudaEvent_t>(start), static_cast<cudaEvent_t>(stop));
}
int s1_host_alloc(void** ptr, size_t bytes) { return cudaHostAlloc(ptr, bytes, cudaHostAllocDefault); }
int s1_host_free(void* ptr) { return cudaFreeHost(ptr); }
int s1_upload_async(void* dst, const void* src, size_t bytes, void* stream) {
    return cudaMemcpyAsync(dst, src, bytes, cudaMemcpyHostToDevice, static_cast<cudaStream_t>(stream));
}
int s1_download_async(void* dst, const void* src, size_t bytes, void* stream) {
    return cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream));
}
int s1_memset_async(void* dst, int value, size_t bytes, void* stream) {
    return cudaMemsetAsync(dst, value, bytes, static_cast<cudaStream_t>(stream));
}
int s1_device_sync(void) { return cudaDeviceSynchronize(); }
int s1_set_dependent_launch(int mode) {
    const int before = s1::dep_launch_switch();
    s1::dep_launch_switch() = mode == 1 || mode == 2 ? mode : 0;
    return before;
}
int s1_mem_info(size_t* free_bytes, size_t* total_bytes) { return cudaMemGetInfo(free_bytes, total_bytes); }

}  // extern "C"
