from .params import BeamSearchParams, SamplingParams
from .sampler import Sampler, request_seed
