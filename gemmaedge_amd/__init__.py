"""gemmaedge_amd — MI355X (gfx950) token-sampling path for GemmaEdge.

The product is the HIP library lib/libgemmaedge_sampler.so with the C ABIs in
include/gemmaedge_sampler.h (sampling), include/gemmaedge_head.h (scoring and
training the answer head), include/gemmaedge_projection.h (a projection with an
adapter for each request) and include/gemmaedge_rules.h (rules on logits), and
the C++ drop-in in include/gemmaedge/sampling.h. This package is its Python bindings
(``sampler``; ``head``, ``projection`` and ``rules``, imported by themselves) and
the synthetic workloads of the benchmark configurations (``workloads``).
"""
from .sampler import (  # noqa: F401
    GE_DTYPE_BF16,
    GE_DTYPE_F32,
    GE_FLAG_NEAR_BOUNDARY,
    GE_FLAG_UNSUPPORTED,
    LIB_PATH,
    SampleArgs,
    SampleParams,
    Sampler,
    SamplerError,
    SamplingConfig,
    available,
    last_error,
    load_library,
    max_top_k,
)
