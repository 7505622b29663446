from .a2c_acktr import A2C_ACKTR
from .adamw import AdamW
from .ppo import PPO
