from dispec_b200.engine.batch import SeqEntry, StepContext, TreeEntry
from dispec_b200.engine.beam import BeamSearchEngine, Hypothesis
from dispec_b200.engine.llm_engine import LLMEngine
from dispec_b200.engine.runner import ModelRunner
from dispec_b200.engine.scheduler import (ContinuousBatchingEngine, Request, Scheduler, State,
                                          StepPlan)
from dispec_b200.engine.speculative import SpeculativeEngine

__all__ = ["SeqEntry", "StepContext", "LLMEngine", "ModelRunner", "ContinuousBatchingEngine",
           "Request", "Scheduler", "State", "StepPlan", "SpeculativeEngine", "TreeEntry",
           "BeamSearchEngine", "Hypothesis"]
