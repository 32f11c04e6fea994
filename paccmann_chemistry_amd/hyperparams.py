"""Factories: same keys as the reference's ``utils/hyperparams.py``, and the
search that a params file names."""
import torch.optim as optim

from .search import (
    BeamSearch, GreedySearch, JointBeamSearch, SamplingSearch
)

SEARCH_FACTORY = {
    'sampling': SamplingSearch,
    'greedy': GreedySearch,
    'beam': BeamSearch,
}

# the searches that ``decoder_search`` can name: the reference's and this one
SEARCHES = dict(SEARCH_FACTORY, joint_beam=JointBeamSearch)


def search_from_params(params):
    """The search of a params file: ``decoder_search`` ('sampling', 'greedy',
    'beam' or 'joint_beam') made with ``temperature``, ``beam_width`` and
    ``top_tokens``, as the training script does it (examples/train_vae.py)."""
    return SEARCHES[params.get('decoder_search', 'sampling')](
        temperature=params.get('temperature', 1.),
        beam_width=params.get('beam_width', 3),
        top_tokens=params.get('top_tokens', 5)
    )


OPTIMIZER_FACTORY = {
    'adadelta': optim.Adadelta,
    'adagrad': optim.Adagrad,
    'adam': optim.Adam,
    'adamax': optim.Adamax,
    'rmsprop': optim.RMSprop,
    'sgd': optim.SGD
}
