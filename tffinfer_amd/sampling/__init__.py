from .params import STRATEGIES, SamplingConfig
from .sampler import Sampler, SeenTokens, TokenLog, allowed_mask, allows_none, uniform_at
