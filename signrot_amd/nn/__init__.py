from .linear import Linear4bit, AsymSymmLinear4bit, GroupLinear4bit
from .quantization import Quantizer, Quantizer8bit, SymQuantizer, AsymQuantizer
from .lora import LoraAdapters
from .hadamard import OnlineHadamard, HadamardQuantizer, fuse_online_hadamard
from .normalization import RMSNorm
from .moe import SignRotMoEBlock
