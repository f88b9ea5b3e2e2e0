from .softmax_xentropy import SoftmaxCrossEntropyLoss  # noqa: F401
from .topk_distillation import SoftmaxTopKDistillationLoss  # noqa: F401
