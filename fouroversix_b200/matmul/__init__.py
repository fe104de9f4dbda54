from .backend import B200MatmulBackend
from .frontend import quantized_matmul
from .grouped import (GroupedQuantizedTensor, GroupLayout, StackedQuantizedTensor, grouped_quantize,
                      grouped_quantized_matmul)
from .weight_only import grouped_weight_only_matmul, weight_only_matmul

__all__ = ["B200MatmulBackend", "GroupLayout", "GroupedQuantizedTensor", "StackedQuantizedTensor",
           "grouped_quantize", "grouped_quantized_matmul", "grouped_weight_only_matmul", "quantized_matmul", "weight_only_matmul"]
