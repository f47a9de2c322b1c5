"""Which kernels a call launches: the call captured in a CUDA graph, and the names of the graph's kernel nodes."""
import re
import warnings

import torch


def kernels_of(call, tmp_path):
    """The mangled names of the kernels that `call` launches, in any order. The call must have run before."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    graph.enable_debug_mode()
    with torch.cuda.graph(graph):
        call()
    path = tmp_path / "graph.dot"
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        graph.debug_dump(str(path))
    return re.findall(r"_Z\w+", path.read_text())
