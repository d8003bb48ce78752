from .acquisition import EI, POI, UCB, UE, PBest, Thompson, shrink_pool
from .base_acq import ei, poi, ucb, ue
from .penalties import compute_penalty
from .pool import ChoiceLogprobs, PoolEviction, choice_logprobs, choice_logprobs_grad, pool_evict, pool_weights

__all__ = ["UCB", "EI", "POI", "UE", "Thompson", "PBest", "shrink_pool", "ei", "ucb", "poi", "ue", "compute_penalty", "choice_logprobs",
           "choice_logprobs_grad", "pool_weights", "pool_evict", "ChoiceLogprobs", "PoolEviction"]
