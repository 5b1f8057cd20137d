"""The draft model around the INT8 tier (mirror of reference ksdraft/model/__init__.py)."""

from .adapters import (AdaptedLinear, adapter_parameters, adapter_state_dict, add_adapters,
                       select_adapters, selected_adapters)
from .block import DraftBlock
from .draft import KSDraftModel
from .generate import draft_block, speculative_step
from .int8_convert import int8_surfaces, to_int8, to_token_channel
from .ks3 import KS3, spine_horner
from .rosa import RosaMixer, _match_payload_sign
from .spine import AdjacentInjection

__all__ = ["KS3", "spine_horner", "RosaMixer", "AdjacentInjection", "DraftBlock",
           "KSDraftModel", "to_int8", "to_token_channel", "int8_surfaces", "_match_payload_sign",
           "AdaptedLinear", "add_adapters", "select_adapters", "selected_adapters", "adapter_parameters", "adapter_state_dict",
           "draft_block", "speculative_step"]
