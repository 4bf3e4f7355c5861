from .lightning_attn2 import (  # noqa: F401
    LightningAttention2,
    LightningAttention2NoDecay,
    lightning_attn2,
    lightning_attn2_no_decay,
    lightning_attn2_parallel,
    la_generic,
    la_dkdv,
    lightning_attn_prefill,
    lightning_attn_decode,
)
from .srmsnorm import SimpleRMSNorm, _SrmsNorm, srmsnorm_sigmoid_gate  # noqa: F401
from .layernorm import LayerNorm, layer_norm, layer_norm_sigmoid_gate  # noqa: F401
from .checkpoint8 import pack_8bit, unpack_8bit  # noqa: F401
