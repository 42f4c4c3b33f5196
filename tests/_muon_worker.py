"""``_sync_worker.py`` with the Muon optimizer: the same options, every rank trains with it."""
import functools

import _sync_worker

_sync_worker.TrainConfig = functools.partial(_sync_worker.TrainConfig, optimizer="muon")

if __name__ == "__main__":
    _sync_worker.main()
