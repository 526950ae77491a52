"""Test package.  Spawned ranks send their results through queues: a tensor travels as a file descriptor that the receiver asks the
sender for, so a rank stays for a moment before it takes down what answers."""
import multiprocessing
import time
from multiprocessing import util

if multiprocessing.current_process().name != "MainProcess":
    util.Finalize(None, time.sleep, args=(2.0,), exitpriority=10)        # ahead of the other finalizers
