// Constant fills as kernels.  A memset recorded into a HIP graph is a node of its own kind, and such nodes have left old
// contents standing in replays after the first; a kernel is replayed like any other.
#include <vector>
#include "common.h"

namespace {

__global__ __launch_bounds__(256) void k_fill(uint32_t *p, uint32_t v, int64_t rows, int64_t cols, int64_t ld) {
    const int64_t total = rows * cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / cols;
        p[r * ld + (i - r * cols)] = v;
    }
}

// 16 bytes a lane; n4 whole quarters, then the rest
__global__ __launch_bounds__(256) void k_fill4(uint32_t *p, uint32_t v, int64_t n) {
    const int64_t n4 = n / 4, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (int64_t i = i0; i < n4; i += (int64_t)gridDim.x * 256) reinterpret_cast<uint4 *>(p)[i] = make_uint4(v, v, v, v);
    if (i0 < n - 4 * n4) p[4 * n4 + i0] = v;
}

}  // namespace

namespace magic {

// (plain launches: the timing brackets of MAGIC_LAUNCH create events, which one caller may not)
int fill_rows(void *p, uint32_t v, int64_t rows, int64_t cols, int64_t ld, hipStream_t stream) {
    if (rows <= 0 || cols <= 0) return MAGIC_OK;
    if (rows == 1 || ld == cols) {
        const int64_t n = rows * cols;
        if ((uintptr_t)p % 16 == 0)
            hipLaunchKernelGGL(k_fill4, dim3(stride_grid(n, 1024)), dim3(256), 0, stream, (uint32_t *)p, v, n);
        else
            hipLaunchKernelGGL(k_fill, dim3(stride_grid(n, 256)), dim3(256), 0, stream, (uint32_t *)p, v, 1, n, n);
    } else {
        hipLaunchKernelGGL(k_fill, dim3(stride_grid(rows * cols, 256)), dim3(256), 0, stream, (uint32_t *)p, v, rows, cols, ld);
    }
    return launch_status();
}

}  // namespace magic

extern "C" int magic_graph_memset_nodes(void *graph, int64_t *count) {
    if (!graph || !count) return MAGIC_ERR_INVALID_ARG;
    size_t n = 0;
    if (hipGraphGetNodes((hipGraph_t)graph, nullptr, &n) != hipSuccess) return MAGIC_ERR_RUNTIME;
    std::vector<hipGraphNode_t> nodes;
    try {
        nodes.resize(n);
    } catch (...) {
        return MAGIC_ERR_RUNTIME;
    }
    if (n > 0 && hipGraphGetNodes((hipGraph_t)graph, nodes.data(), &n) != hipSuccess) return MAGIC_ERR_RUNTIME;
    *count = 0;
    for (size_t i = 0; i < n; ++i) {
        hipGraphNodeType t;
        if (hipGraphNodeGetType(nodes[i], &t) != hipSuccess) return MAGIC_ERR_RUNTIME;
        *count += t == hipGraphNodeTypeMemset;
    }
    return MAGIC_OK;
}
