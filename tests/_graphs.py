"""What a call launches, read from a graph that captures it."""

from __future__ import annotations

import torch


def kernels_of(call) -> list[str]:
    """Names (as the linker has them) of the kernels that call() launches, which is captured and not run."""
    from cuda.bindings import driver

    def ok(result):
        assert int(result[0]) == 0, result[0]
        return result[1:]

    call()  # what a first call sets up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    count = ok(driver.cuGraphGetNodes(raw, 0))[1]
    names = []
    for node in ok(driver.cuGraphGetNodes(raw, count))[0]:
        if ok(driver.cuGraphNodeGetType(node))[0] == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            p = ok(driver.cuGraphKernelNodeGetParams(node))[0]
            names.append(ok(driver.cuFuncGetName(p.func) if int(p.func) else driver.cuKernelGetName(p.kern))[0].decode())
    return names
