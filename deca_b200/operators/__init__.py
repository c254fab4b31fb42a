from .Op import Operator
from .GEMMTC import GEMMTC
from .FlashAttention import FlashAttention
from .Rowwise import RowwiseOperator, TOLERANCE
from .Softmax import Softmax
from .RMSNorm import RMSNorm
from .AddRMSNorm import AddRMSNorm
from .Rotary import Rotary, RotaryAppend
from .Paged import PagedAttention, PagedStep, PagedStepResult

__all__ = ["Operator", "GEMMTC", "FlashAttention", "RowwiseOperator", "Softmax", "RMSNorm", "TOLERANCE",
           "AddRMSNorm", "Rotary", "RotaryAppend", "PagedAttention", "PagedStep", "PagedStepResult"]
