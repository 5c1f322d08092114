"""A queue between processes whose tensors travel by value.

torch sends a CPU tensor as a handle that its sender has to serve until it is
taken.  A worker that ends right after its put() leaves the receiver a handle
that nobody serves (EOFError, ConnectionResetError, FileNotFoundError)."""

import pickle
from multiprocessing.queues import SimpleQueue


class ValueQueue(SimpleQueue):
    def put(self, obj):
        super().put(pickle.dumps(obj))

    def get(self):
        return pickle.loads(super().get())
