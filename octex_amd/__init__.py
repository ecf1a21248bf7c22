"""octex for MI355X: approximate k-nearest-neighbor search by E8-lattice cell lists (cuvs::neighbors::octex),
with every search step a hand-written HIP kernel for gfx950.

    import octex_amd as octex
    index = octex.load("index_dir")        # or octex.build(xb, "index_dir")
    D, I = index.search(xq, k=10)          # (distances, neighbors), nearest first

Operators on rows of scores, for models that make the queries or read the neighbors (octex_amd/scores.py):
quantize_rows, int8_scores, log_probs, log_probs_backward, distill, distill_backward, distill_step.

Drop-ins: `from octex_amd import cuvs as cagra` (cuvs.neighbors.cagra calls) and `from octex_amd import faiss`
(Faiss GPU index calls).
"""

from .index import Index, build, build_in_memory, load
from .scores import (LogProbs, distill, distill_backward, distill_step, int8_scores, log_probs, log_probs_backward,
                     quantize_rows)

__version__ = "0.1.0"
__all__ = ["Index", "LogProbs", "build", "build_in_memory", "distill", "distill_backward", "distill_step", "int8_scores",
           "load", "log_probs", "log_probs_backward", "quantize_rows", "__version__"]
